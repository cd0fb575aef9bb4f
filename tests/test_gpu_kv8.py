"""-m gpu: the 8-bit key / value cache (modules.kv8_cache.KV8Cache) against its definition in 64 bits.

Tolerances, fixed before the first run.  u(t) = finfo(t).eps / 2 is one rounding to t.

  store / load   the codes are whole numbers by the format's rule, computed here with the same 32-bit product: equal; a value is
                 code * scale, the scale one rounding and the product one (and one to the output type): 3 u(f32) (+ u(bf16))
  attention      scores: exact products of <= 8 x 22-bit numbers summed in f32; |error of a score| <= 2^-17 for |score| <= ~40
                 (f32 sums of 128 terms, 2^-24 each, and the f32 factor), which is a relative error of 2^-17 of a probability;
                 probabilities: f32 results take a pair of f16 (2^-22), bf16 ones a single f16 (2^-12 at most); sums in f32 over
                 n tokens: the probabilities are positive, so sum |p v| / sum p <= max |v|, and everything is relative to max |v|:
                 f32: 2^-15 max |v|      bf16: (2^-11 + u(bf16)) max |v|   (u(bf16) = 2^-8 relative to the result <= max |v|)
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BLK = 64
DT = {'f32': torch.float32, 'bf16': torch.bfloat16}


@pytest.fixture(scope='module')
def KV8Cache():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from audiocraft_amd.modules.kv8_cache import KV8Cache
    return KV8Cache


@pytest.fixture(params=['own rows', 'among many rows'])
def AnyCache(request, KV8Cache):
    """The cache, or the same rows in front of 800 empty ones: the grid is then large, and prompts take the form for that."""
    if request.param == 'own rows':
        return KV8Cache

    class Among(KV8Cache):
        extra = 800

        def __init__(self, rows, *a, **kw):
            super().__init__(rows + self.extra, *a, **kw)

        def more(self, t):
            if t is None or t.shape[0] == self.rows:
                return t
            out = t.new_zeros(self.rows, *t.shape[1:])
            out[:t.shape[0]] = t
            return out

        def store(self, k, v, start=None, n=None):
            n = torch.full((k.shape[0],), k.shape[1], dtype=torch.int32, device='cuda') if n is None else n
            super().store(self.more(k), self.more(v), self.more(start), self.more(n))

        def attend(self, q, lens, causal=True, past_context=0, q_lens=None, starts=None):
            return super().attend(self.more(q), self.more(lens), causal, past_context, self.more(q_lens), self.more(starts))[:q.shape[0]]

        def decode(self, q, k, v, lens, past_context=0, starts=None):
            return super().decode(self.more(q), self.more(k), self.more(v), self.more(lens), past_context, self.more(starts))[:q.shape[0]]
    return Among


# ------------------------------------------------------------------------------------------ the definition

def quantised(block):
    """[64, ..] f32 of one (block, head) -> the values its codes stand for, f64 (codes by the format's 32-bit rule)."""
    amax = block.abs().max()
    if not torch.isfinite(block).all():
        return torch.full_like(block, math.nan, dtype=torch.float64)
    if amax < 2.0 ** -120:
        return torch.zeros_like(block, dtype=torch.float64)
    codes = torch.round(block * (torch.tensor(127.0) / amax))
    return codes.double() * (amax / torch.tensor(127.0)).double()


def held(x):
    """[n, H, hd] f32 (as rounded to the cache's type) -> what the cache holds of it, f64."""
    out = x.double().clone()
    for b in range(max(len(x) - 1, 0) // BLK):
        for h in range(x.shape[1]):
            out[b * BLK:(b + 1) * BLK, h] = quantised(x[b * BLK:(b + 1) * BLK, h])
    return out


def attention(q, k, v, causal, qlen, past, start):
    """q [S, Hq, hd], k / v [n, H, hd] f64 -> [S, Hq, hd]; tokens that a query does not see do not enter at all."""
    S, Hq, hd = q.shape
    n, H = k.shape[:2]
    out = torch.zeros(S, Hq, hd, dtype=torch.float64)
    for i in range(qlen):
        hi = n - qlen + i + 1 if causal else n
        lo = max(start, hi - 1 - past) if causal and past else start
        if hi <= lo:
            continue
        for h in range(Hq):
            s = k[lo:hi, h * H // Hq] @ q[i, h] / math.sqrt(hd)
            out[i, h] = torch.softmax(s, 0) @ v[lo:hi, h * H // Hq]
    return out


def tol(dt, vmax):
    return (2.0 ** -15 if dt == torch.float32 else 2.0 ** -11 + 2.0 ** -8) * vmax


def make(R, n, H, hd, dt, seed, dev='cuda'):
    g = torch.Generator().manual_seed(seed)
    k = (torch.randn(R, n, H, hd, generator=g) + torch.randn(1, 1, H, hd, generator=g)).to(dt)
    v = torch.randn(R, n, H, hd, generator=g).to(dt)
    return k, v


def words(*xs):
    return torch.tensor(xs, dtype=torch.int32, device='cuda')


def filled(KV8Cache, lens, H, hd, dt, seed, capacity=None):
    R, n = len(lens), max(max(lens), 1)
    k, v = make(R, n, H, hd, dt, seed)
    c = KV8Cache(R, H, hd, capacity or n + 1, dtype=dt)
    c.store(k.cuda(), v.cuda(), words(*[0] * R), words(*lens))
    return c, k, v


# ------------------------------------------------------------------------------------------ store / load

@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('hd', [16, 32, 64, 128])
@pytest.mark.parametrize('lens', [[1], [0, 63, 64], [65, 128, 129, 200]])
def test_store_load(KV8Cache, dt, hd, lens):
    dt = DT[dt]
    c, k, v = filled(KV8Cache, lens, 3, hd, dt, hd + len(lens), capacity=256)
    for out_dt in (torch.float32, torch.bfloat16):
        gk, gv = (t.cpu() for t in c.load(words(*lens), 210, dtype=out_dt))
        for r, n in enumerate(lens):
            for got, x in ((gk, k), (gv, v)):
                ref = held(x[r, :n].float()).permute(1, 0, 2)
                rel = 3 * 2.0 ** -24 + (2.0 ** -8 if out_dt == torch.bfloat16 else 0)
                assert ((got[r, :, :n].double() - ref).abs() <= rel * ref.abs()).all()
                assert (got[r, :, n:] == 0).all()


@pytest.mark.parametrize('chunks', [[1] * 70, [63, 1, 1], [30, 40, 100], [64, 64], [5, 200, 3], [129, 1]])
def test_store_in_chunks_equals_store_at_once(KV8Cache, chunks):
    n = sum(chunks)
    k, v = make(2, n, 2, 32, torch.bfloat16, n)
    whole, parts = (KV8Cache(2, 2, 32, n) for _ in range(2))
    zero = words(0, 0)
    whole.store(k.cuda(), v.cuda(), zero)
    at = 0
    for m in chunks:
        parts.store(k[:, at:at + m].cuda(), v[:, at:at + m].cuda(), words(at, at))
        at += m
    for a, b in zip(whole.load(words(n, n)), parts.load(words(n, n))):
        assert torch.equal(a, b)
    for name in ('k_codes', 'v_codes', 'k_scale', 'v_scale'):
        assert torch.equal(getattr(whole, name), getattr(parts, name))


def test_store_reads_no_padding_and_leaves_other_rows(KV8Cache):
    c, k, v = filled(KV8Cache, [100, 70, 64], 2, 64, torch.float32, 3, capacity=256)
    before = [t.clone() for t in (c.k_codes, c.v_codes, c.k_scale, c.v_scale, c.k_tail, c.v_tail)]
    x = torch.full((3, 80, 2, 64), math.nan)
    x[1, :30] = 1.0
    c.store(x.cuda(), x.cuda(), words(100, 70, 64), words(0, 30, 0))
    for t, b in zip((c.k_codes, c.v_codes, c.k_scale, c.v_scale, c.k_tail, c.v_tail), before):
        assert torch.equal(t[0], b[0]) and torch.equal(t[2], b[2])
    gk, _ = c.load(words(100, 100, 64), 128)
    assert torch.isfinite(gk).all() and (gk[1, :, 70:100] == 1.0).all() and (gk[:, :, 100:] == 0).all()


def test_store_past_the_capacity_is_dropped(KV8Cache):
    k, v = make(2, 100, 1, 16, torch.float32, 5)
    c = KV8Cache(2, 1, 16, 64)
    assert c.capacity == 64
    c.store(k.cuda(), v.cuda(), words(0, 64))       # row 0: 100 tokens into 64 places; row 1 is full already
    gk, _ = c.load(words(1000, 64))
    assert torch.equal(gk[0, 0].cpu(), k[0, :64, 0].to(torch.bfloat16).float())   # the newest block: as stored
    assert (gk[1] == 0).all()


@pytest.mark.parametrize('strides', ['packed', 'heads_first', 'expanded'])
def test_store_strides(KV8Cache, strides):
    R, n, H, hd = 2, 130, 4, 64
    k, v = make(R, n, H, hd, torch.bfloat16, 11)
    if strides == 'packed':           # slices of one projection, odd offset
        buf = torch.zeros(R, n, 3 * H * hd + 1, dtype=torch.bfloat16, device='cuda')
        kk, vv = buf[..., 1 + H * hd:1 + 2 * H * hd].unflatten(-1, (H, hd)), buf[..., 1 + 2 * H * hd:].unflatten(-1, (H, hd))
        kk.copy_(k)
        vv.copy_(v)
    elif strides == 'heads_first':
        kk, vv = (t.cuda().permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (k, v))
    else:                              # the same head for all
        k, v = (t[:, :, :1].expand(R, n, H, hd) for t in (k, v))
        kk, vv = (t[:, :, :1].cuda().expand(R, n, H, hd) for t in (k, v))
    c = KV8Cache(R, H, hd, n)
    c.store(kk, vv, words(0, 0))
    for got, x in zip(c.load(words(n, n), n), (k, v)):
        for r in range(R):
            ref = held(x[r].float()).permute(1, 0, 2)
            assert ((got[r].cpu().double() - ref).abs() <= 3 * 2.0 ** -24 * ref.abs()).all()


def test_block_scales_special_values(KV8Cache):
    """Zero blocks, tiny ones, the largest numbers, and a block poisoned by one NaN or infinity."""
    x = torch.zeros(6, 65, 1, 16)
    x[1, :64] = 1e-38
    x[2, :64, 0, 0] = 3.0e38
    x[2, 5, 0, 3] = -3.4e38
    x[3, 7, 0, 2] = math.nan
    x[4, 7, 0, 2] = -math.inf
    x[5, :64] = 2.0 ** -119
    c = KV8Cache(6, 1, 16, 128, dtype=torch.float32)
    c.store(x.cuda(), x.cuda(), words(*[0] * 6))
    gk, gv = (t.cpu() for t in c.load(words(*[65] * 6), 65))
    for got in (gk, gv):
        assert (got[0] == 0).all() and (got[1] == 0).all()
        ref = held(x[2]).permute(1, 0, 2)
        assert ((got[2].double() - ref).abs() <= 3 * 2.0 ** -24 * ref.abs()).all()
        for r in (3, 4):
            assert got[r, 0, :64].isnan().all() and (got[r, 0, 64] == 0).all()
        assert ((got[5, 0, :64].double() - 2.0 ** -119).abs() <= 3 * 2.0 ** -24 * 2.0 ** -119).all()


# ------------------------------------------------------------------------------------------ attention

def check(got, ref, dt, vmax):
    err = (got.cpu().double() - ref).abs().max().item()
    assert err <= tol(dt, vmax), (err, tol(dt, vmax))


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('H,G,hd', [(3, 1, 64), (2, 4, 128), (1, 17, 32), (2, 3, 16)])
@pytest.mark.parametrize('lens', [[0], [1, 62, 63, 64], [127, 128, 300], [2100, 700]])
def test_decode(KV8Cache, dt, H, G, hd, lens):
    dt, R = DT[dt], len(lens)
    c, k, v = filled(KV8Cache, lens, H, hd, dt, 7 * R + hd, capacity=max(lens) + 1)
    g = torch.Generator().manual_seed(hd + G)
    q = torch.randn(R, H * G, hd, generator=g).to(dt)
    k1, v1 = torch.randn(R, H, hd, generator=g).to(dt), torch.randn(R, H, hd, generator=g).to(dt)
    got = c.decode(q.cuda(), k1.cuda(), v1.cuda(), words(*lens))
    after = c.load(words(*[n + 1 for n in lens]), max(lens) + 1)
    for r, n in enumerate(lens):
        kr, vr = (torch.cat([x[r, :n], x1[r:r + 1]]).float() for x, x1 in ((k, k1), (v, v1)))
        ref = attention(q[r:r + 1].double(), held(kr), held(vr), True, 1, 0, 0)
        check(got[r:r + 1], ref, dt, vr.abs().max().item())
        for t, x in zip(after, (kr, vr)):       # the token is stored, and a block it completes is quantised
            ref = held(x).permute(1, 0, 2)
            assert ((t[r, :, :n + 1].cpu().double() - ref).abs() <= 3 * 2.0 ** -24 * ref.abs()).all()


def test_decode_token_by_token_equals_store(KV8Cache):
    """130 decode steps leave the cache that one store leaves."""
    R, H, hd, n = 2, 2, 64, 130
    k, v = make(R, n, H, hd, torch.float32, 1)
    a, b = (KV8Cache(R, H, hd, n) for _ in range(2))
    a.store(k.cuda(), v.cuda(), words(0, 0))
    q = torch.randn(R, H, hd, device='cuda')
    for t in range(n):
        b.decode(q, k[:, t].cuda(), v[:, t].cuda(), words(t, t))
    for x, y in zip(a.load(words(n, n)), b.load(words(n, n))):
        assert torch.equal(x, y)
    for name in ('k_codes', 'v_codes', 'k_scale', 'v_scale'):
        assert torch.equal(getattr(a, name), getattr(b, name))


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('G,lens', [(65, [127, 3]), (80, [63, 0]), (130, [700, 65])])
def test_decode_with_many_heads_on_one(KV8Cache, dt, G, lens):
    """More query heads per cache head than one workgroup's column tile times four: the token is stored all the same."""
    dt, hd = DT[dt], 64
    c, k, v = filled(KV8Cache, lens, 1, hd, dt, G, capacity=max(lens) + 1)
    g = torch.Generator().manual_seed(G)
    q = torch.randn(2, G, hd, generator=g).to(dt)
    k1, v1 = torch.randn(2, 1, hd, generator=g).to(dt), torch.randn(2, 1, hd, generator=g).to(dt)
    got = c.decode(q.cuda(), k1.cuda(), v1.cuda(), words(*lens))
    after = c.load(words(*[n + 1 for n in lens]), max(lens) + 1)
    for r, n in enumerate(lens):
        kr, vr = (torch.cat([x[r, :n], x1[r:r + 1]]).float() for x, x1 in ((k, k1), (v, v1)))
        check(got[r:r + 1], attention(q[r:r + 1].double(), held(kr), held(vr), True, 1, 0, 0), dt, vr.abs().max().item())
        for t, x in zip(after, (kr, vr)):
            ref = held(x).permute(1, 0, 2)
            assert ((t[r, :, :n + 1].cpu().double() - ref).abs() <= 3 * 2.0 ** -24 * ref.abs()).all()


def test_a_cache_is_not_copied_as_an_object(KV8Cache):
    import copy
    c = KV8Cache(1, 1, 16, 64)
    for f in (copy.copy, copy.deepcopy):
        with pytest.raises(TypeError, match="load"):
            f(c)


def test_decode_on_a_full_row_drops_the_token(KV8Cache):
    c, k, v = filled(KV8Cache, [128, 100], 2, 64, torch.float32, 2, capacity=128)
    before = [t[0].clone() for t in (c.k_codes, c.v_codes, c.k_tail, c.v_tail, c.k_scale)]
    x = torch.full((2, 2, 64), 9.0, device='cuda')
    q = torch.randn(2, 2, 64, device='cuda')
    got = c.decode(q, x, x, words(128, 100))
    for t, b in zip((c.k_codes, c.v_codes, c.k_tail, c.v_tail, c.k_scale), before):
        assert torch.equal(t[0], b)
    ref = attention(q[:1].cpu().double(), held(k[0]), held(v[0]), True, 1, 0, 0)
    check(got[:1], ref, torch.float32, v.abs().max().item())


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('causal,past', [(True, 0), (True, 1), (True, 100), (False, 0)])
@pytest.mark.parametrize('H,G,hd,S', [(2, 1, 64, 1), (1, 4, 64, 5), (2, 2, 128, 70), (1, 3, 32, 150), (3, 1, 16, 33), (1, 1, 64, 200)])
def test_attend(AnyCache, dt, causal, past, H, G, hd, S):
    dt = DT[dt]
    lens = [max(S, 1), 257, 64, 130, 0, 40]
    q_lens = [min(S, n) if causal else S for n in lens]
    q_lens[1] = min(S, 3)                              # a padded batch
    starts = [0, 70, 0, 0, 0, 1000]                    # left padding; the last row sees nothing at all
    R = len(lens)
    c, k, v = filled(AnyCache, lens, H, hd, dt, S + hd)
    g = torch.Generator().manual_seed(S)
    q = torch.randn(R, S, H * G, hd, generator=g).to(dt)
    got = c.attend(q.cuda(), words(*lens), causal=causal, past_context=past, q_lens=words(*q_lens), starts=words(*starts))
    for r, n in enumerate(lens):
        kr, vr = (held(x[r, :n].float()) for x in (k, v))
        ref = attention(q[r].double(), kr, vr, causal, q_lens[r], past, starts[r])
        check(got[r], ref, dt, 1e-30 if n == 0 else v[r].float().abs().max().item())
        seen = [i for i in range(S) if i < q_lens[r] and (n - q_lens[r] + i + 1 if causal else n) > starts[r]]
        dead = [i for i in range(S) if i not in seen]
        assert (got[r, dead] == 0).all()


@pytest.mark.parametrize('H,G,hd,S', [(1, 1, 64, 64), (1, 1, 64, 65), (1, 1, 128, 64), (1, 1, 128, 65), (1, 33, 16, 2), (1, 13, 32, 5), (2, 1, 64, 129)])
@pytest.mark.parametrize('dt', ['f32', 'bf16'])
def test_attend_where_the_forms_change(AnyCache, dt, H, G, hd, S):
    """Whole column tiles and one column more, of a workgroup and of a wave."""
    dt, lens = DT[dt], [190, S, 0]
    c, k, v = filled(AnyCache, lens, H, hd, dt, S + G)
    q = torch.randn(3, S, H * G, hd, generator=torch.Generator().manual_seed(S)).to(dt)
    got = c.attend(q.cuda(), words(*lens))
    for r, n in enumerate(lens):
        kr, vr = k[r, :n].float(), v[r, :n].float()
        check(got[r], attention(q[r].double(), held(kr), held(vr), True, S, 0, 0), dt, max(vr.abs().max().item() if n else 0, 1e-30))


@pytest.mark.parametrize('H', [384, 200])
@pytest.mark.parametrize('causal,past', [(True, 0), (True, 90), (False, 0)])
def test_attend_on_a_full_grid(KV8Cache, causal, past, H):
    """Enough heads that a wave takes two column tiles, and enough for the prompt form; the queries heads first in memory."""
    hd, S, lens = 64, 70, [333, 64]
    c, k, v = filled(KV8Cache, lens, H, hd, torch.bfloat16, 41)
    q = torch.randn(2, S, H, hd, generator=torch.Generator().manual_seed(42)).bfloat16()
    starts, q_lens = [0, 9], [S, 50]
    got = c.attend(q.transpose(1, 2).contiguous().cuda().transpose(1, 2), words(*lens), causal, past, words(*q_lens), words(*starts))
    for r, n in enumerate(lens):
        kr, vr = k[r, :n].float(), v[r, :n].float()
        s = torch.einsum('shd,thd->hst', q[r].double(), held(kr)) / math.sqrt(hd)
        i, t = (n - q_lens[r] + torch.arange(S))[:, None], torch.arange(n)[None]
        seen = (t >= starts[r]) & (torch.arange(S)[:, None] < q_lens[r])
        if causal:
            seen = seen & (t <= i) & ((t >= i - past) if past else (t >= 0))
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
        check(got[r], torch.einsum('hst,thd->shd', p, held(vr)), torch.bfloat16, vr.abs().max().item())


def test_attend_long_context_is_split_and_joined(AnyCache):
    """One row, 9000 tokens: the split form; the same call again gives the same bits."""
    c, k, v = filled(AnyCache, [9000, 70], 2, 64, torch.float32, 4)
    q = torch.randn(2, 2, 4, 64, generator=torch.Generator().manual_seed(0))
    got = c.attend(q.cuda(), words(9000, 70))
    for r, n in enumerate((9000, 70)):
        check(got[r], attention(q[r].double(), held(k[r, :n]), held(v[r, :n]), True, 2, 0, 0), torch.float32, v.abs().max().item())
    for _ in range(3):
        assert torch.equal(got, c.attend(q.cuda(), words(9000, 70)))


def test_q_longer_than_the_row(AnyCache):
    """Causal queries that would sit before the row's first token see nothing."""
    c, k, v = filled(AnyCache, [3, 80], 1, 32, torch.float32, 8)
    q = torch.randn(2, 90, 1, 32, generator=torch.Generator().manual_seed(2))
    got = c.attend(q.cuda(), words(3, 80))
    for r, n in enumerate((3, 80)):
        assert (got[r, :90 - n] == 0).all()
        ref = attention(q[r, 90 - n:].double(), held(k[r, :n]), held(v[r, :n]), True, n, 0, 0)
        check(got[r, 90 - n:], ref, torch.float32, v.abs().max().item())


@pytest.mark.parametrize('S', [1, 100])
def test_what_is_not_seen_does_not_matter(AnyCache, S):
    """NaN and infinity in tail places past the row's length, in tokens before `starts`, and (causal) in later tokens."""
    n = 150
    k, v = make(1, n, 2, 64, torch.float32, 6)
    c, d = (AnyCache(1, 2, 64, 256, dtype=torch.float32) for _ in range(2))
    c.store(k.cuda(), v.cuda(), words(0))
    kb, vb = k.clone(), v.clone()
    kb[:, :64], vb[:, :64] = math.nan, math.inf         # a whole block before `starts`
    kb[:, 149], vb[:, 149, :, 5] = math.nan, -math.inf  # the newest token: seen by the last query alone
    d.store(kb.cuda(), vb.cuda(), words(0))
    d.k_tail[:, :, 22:] = math.nan                      # never reached
    d.v_tail[:, :, 22:] = math.nan
    q = torch.randn(1, S, 2, 64, device='cuda')
    a, b = (x.attend(q, words(n), starts=words(64)) for x in (c, d))
    assert torch.equal(a[:, :-1], b[:, :-1]) and torch.isfinite(b[:, :-1]).all()
    assert b[:, -1].isnan().all()
    got = d.attend(q, words(149), starts=words(64))
    assert torch.isfinite(got).all()


def test_queries_with_special_values(AnyCache):
    c, k, v = filled(AnyCache, [200], 1, 64, torch.float32, 9)
    q = torch.randn(1, 20, 1, 64, generator=torch.Generator().manual_seed(3))
    q[0, 3, 0, 5] = math.nan
    q[0, 4, 0, 5] = math.inf
    q[0, 5] = 0
    q[0, 6] *= 1e-30
    q[0, 7] *= 1e-42
    q[0, 8] = 1e30 * torch.sign(q[0, 8])              # one token takes everything
    got = c.attend(q.cuda(), words(200), causal=False).cpu()
    assert got[0, 3:5].isnan().all()
    live = [i for i in range(20) if i not in (3, 4)]
    ref = attention(q[0, live].double(), held(k[0]), held(v[0]), False, len(live), 0, 0)
    check(got[0, live], ref, torch.float32, v.abs().max().item())


def test_large_scores_and_flat_ones(AnyCache):
    """Scores of +-900 (one token takes all, far tokens underflow) and exactly equal scores over a long row."""
    n = 3000
    k, v = make(1, n, 1, 64, torch.float32, 10)
    c = AnyCache(1, 1, 64, n, dtype=torch.float32)
    c.store(k.cuda(), v.cuda(), words(0))
    q = torch.stack([100.0 * torch.randn(64, generator=torch.Generator().manual_seed(1)), torch.zeros(64)]).view(1, 2, 1, 64)
    got = c.attend(q.cuda(), words(n), causal=False)
    ref = attention(q[0].double(), held(k[0]), held(v[0]), False, 2, 0, 0)
    # scores of ~10^3 in f32: 2^-24 * 10^3 * a few terms of error each instead of the 2^-17 of ordinary ones
    assert (got[0, 0].cpu().double() - ref[0]).abs().max() <= 2.0 ** -11 * v.abs().max()
    check(got[0, 1], ref[1], torch.float32, v.abs().max().item())


@pytest.mark.parametrize('S', [1, 100])
@pytest.mark.parametrize('order', ['falling', 'rising', 'mixed'])
def test_blocks_of_very_different_size(AnyCache, S, order):
    """Values from 1e-25 to 1e10 from block to block, keys from 1e-30 to 1: the queries look at the small ones.

    The size of a result is sum p |v|, far below the largest value held: 2^-15 of that, and what f16 drops of p (n * 2^-33 of the
    largest value a query gives weight to: the large blocks have p < 2^-40 by their keys)."""
    n, hd = 64 * 8 + 10, 64
    k, v = make(1, n, 1, hd, torch.float32, 15)
    size = [1e10, 1e-25, 1.0, 1e-12, 1e-3, 1e5, 1e-20, 1e-7, 1e-15]
    if order != 'mixed':
        size = sorted(size, reverse=order == 'falling')
    q = torch.randn(1, S, 1, hd, generator=torch.Generator().manual_seed(7))
    q[..., 0] = 1.0
    for b, s in enumerate(size):
        v[:, b * BLK:(b + 1) * BLK] *= s
        k[:, b * BLK:(b + 1) * BLK] *= (0.05 if s < 1e-6 else 0.5)
        if s > 1e-6:
            k[:, b * BLK:(b + 1) * BLK, :, 0] = -400.0       # score -50: p < 1e-20 beside the small blocks
    if order == 'mixed':
        k[:, 3 * BLK:4 * BLK] *= 1e-30
    c = AnyCache(1, 1, hd, n, dtype=torch.float32)
    c.store(k.cuda(), v.cuda())
    got = c.attend(q.cuda(), words(n), causal=False).cpu().double()
    kh, vh = held(k[0]), held(v[0])
    for i in range(S):
        p = torch.softmax(kh[:, 0] @ q[0, i, 0].double() / math.sqrt(hd), 0)
        err = (got[0, i, 0] - p @ vh[:, 0]).abs()
        bound = 2.0 ** -15 * (p @ vh[:, 0].abs()) + n * 2.0 ** -33 * vh[:, 0].abs().amax(0) * 1e-17
        assert (err <= bound).all(), (i, (err / bound).max().item())


@pytest.mark.parametrize('S', [1, 60])
@pytest.mark.parametrize('scale', [1e-30, 1e30])
def test_tiny_and_huge_products(AnyCache, S, scale):
    """Keys and queries of 1e-30 each: every score is 0 in f32, the result the mean; values of 1e30: f32's range holds."""
    n = 300
    k, v = make(1, n, 1, 64, torch.float32, 16)
    k, v = (k * 1e-30, v) if scale < 1 else (k, v * 1e30)
    q = torch.randn(1, S, 1, 64, generator=torch.Generator().manual_seed(8)) * (1e-30 if scale < 1 else 1)
    c = AnyCache(1, 1, 64, n, dtype=torch.float32)
    c.store(k.cuda(), v.cuda())
    for starts in (None, words(70)):
        got = c.attend(q.cuda(), words(n), causal=False, starts=starts)
        ref = attention(q[0].double(), held(k[0]), held(v[0]), False, S, 0, 0 if starts is None else 70)
        check(got[0], ref, torch.float32, v.abs().max().item())


@pytest.mark.parametrize('S', [1, 40])
def test_query_strides(AnyCache, S):
    c, k, v = filled(AnyCache, [100, 90], 2, 64, torch.bfloat16, 12)
    q = torch.randn(2, S, 4, 64, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    want = c.attend(q, words(100, 90))
    packed = torch.zeros(2, S, 4 * 64 * 3 + 1, device='cuda', dtype=torch.bfloat16)
    view = packed[..., 1:257].unflatten(-1, (4, 64))
    view.copy_(q)
    assert torch.equal(c.attend(view, words(100, 90)), want)
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(c.attend(heads_first, words(100, 90)), want)
    assert torch.equal(c.attend(q.transpose(2, 3).contiguous().transpose(2, 3), words(100, 90)), want)


# ------------------------------------------------------------------------------------------ as it is used

def test_a_generation_captured_and_replayed(KV8Cache):
    """Prompt, then decode steps as one captured graph whose lengths advance on the device, against the same steps run eagerly;
    eager work and other graphs between the replays."""
    R, H, hd, P, T = 3, 2, 64, 60, 12
    k, v = make(R, P + T, H, hd, torch.float32, 20)
    k, v = k.cuda(), v.cuda()
    qs = torch.randn(T, R, 2 * H, hd, device='cuda', generator=torch.Generator(device='cuda').manual_seed(1))
    lens0 = words(P, P - 5, P - 10)

    def begin(cache):
        cache.store(k[:, :P], v[:, :P], words(0, 0, 0), lens0)

    eager = KV8Cache(R, H, hd, P + T + 1)
    begin(eager)
    lens = lens0.clone()
    want = []
    for t in range(T):
        want.append(eager.decode(qs[t], k[:, P + t], v[:, P + t], lens).clone())
        lens += 1

    graphs = []
    for _ in range(2):                       # two graphs, each with a cache of its own
        cache = KV8Cache(R, H, hd, P + T + 1)
        begin(cache)
        st = dict(q=qs[0].clone(), k=k[:, P].clone(), v=v[:, P].clone(), lens=lens0.clone(), cache=cache)
        cache.decode(st['q'], st['k'], st['v'], st['lens'])     # warm up (idempotent: the length has not advanced)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            st['out'] = cache.decode(st['q'], st['k'], st['v'], st['lens'])
            st['lens'] += 1
        st['lens'].copy_(lens0)
        graphs.append((g, st))
    for t in range(T):
        for g, st in graphs:
            st['q'].copy_(qs[t])
            st['k'].copy_(k[:, P + t])
            st['v'].copy_(v[:, P + t])
            g.replay()
            torch.randn(1000, device='cuda').sum()
            torch.cuda.synchronize()
            assert torch.equal(st['out'], want[t]), t
    for g, st in graphs:
        assert torch.equal(st['lens'], lens)
        for a, b in zip(st['cache'].load(lens), eager.load(lens)):
            assert torch.equal(a, b)


def test_tiled_output_and_one_length_word(KV8Cache):
    """The form the LM's decode step calls: the new token already in the tail, one length word for all rows, f32 queries, the
    result as the next GEMM's tiled bf16 operand at a column offset; the block that the token completes is quantised."""
    import ctypes
    from audiocraft_amd import _C
    R, H, hd, n = 5, 3, 64, 128
    k, v = make(R, n, H, hd, torch.bfloat16, 30)
    whole, c = KV8Cache(R, H, hd, n), KV8Cache(R, H, hd, n)
    whole.store(k.cuda(), v.cuda())
    c.store(k[:, :n - 1].cuda(), v[:, :n - 1].cuda())
    c.k_tail[:, :, 63], c.v_tail[:, :, 63] = k[:, n - 1].cuda(), v[:, n - 1].cuda()
    q = torch.randn(R, H * hd, generator=torch.Generator().manual_seed(5))
    qd, pos, d = q.cuda(), words(n - 1), H * hd
    out = _C.tiled_activation_buffer(R, 2 * d, torch.bfloat16, 'cuda')
    desc = _C.KV8AttnDesc(q=qd.data_ptr(), q_dtype=_C.F32, q_row=d, q_head=hd, S=1, Hq=H, len=pos.data_ptr(), len_stride=0, len_bias=1,
                          causal=1, complete=1, out=out.data_ptr(), out_mode=_C.OUT_TILED, out_dtype=_C.BF16, out_rbs=2 * d // 32, out_col0=d)
    _C.check(_C._kv8_attn(ctypes.byref(c.desc), ctypes.byref(desc), _C.stream()), 'acmi_kv8_attn')
    got = _C.untile_matrix(out, R, 2 * d)
    assert (got[:, :d] == 0).all()
    for r in range(R):
        ref = attention(q[r].view(1, H, hd).double(), held(k[r].float()), held(v[r].float()), True, 1, 0, 0)
        check(got[r, d:].view(1, H, hd), ref, torch.bfloat16, v[r].float().abs().max().item())
    for name in ('k_codes', 'v_codes', 'k_scale', 'v_scale'):
        assert torch.equal(getattr(c, name), getattr(whole, name))


def test_positions_past_32_bit_offsets(KV8Cache):
    """Row 1 begins past 2^31 bytes, its newest tokens lie 2^31 bytes further on."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    hd, start, n, past = 128, 16999040, 200, 100
    c = KV8Cache(2, 1, hd, 17000000)
    k, v = make(1, n, 1, hd, torch.float32, 50)
    both = [torch.cat([x, x]).cuda() for x in (k, v)]
    c.store(*both, words(0, start), words(0, n))
    q = torch.randn(2, 70, 1, hd, generator=torch.Generator().manual_seed(51))
    kr, vr = k[0].bfloat16().float(), v[0].bfloat16().float()
    for S in (3, 70):
        got = c.attend(q[:, :S].cuda(), words(0, start + n), past_context=past)
        assert (got[0] == 0).all()
        check(got[1], attention(q[1, :S].double(), held(kr), held(vr), True, S, past, 0), torch.float32, vr.abs().max().item())
    k1 = torch.randn(2, 1, hd, generator=torch.Generator().manual_seed(52))
    got = c.decode(q[:, 0].cuda(), k1.cuda(), k1.cuda(), words(0, start + n), past)
    kr, vr = (torch.cat([x, k1[1:].bfloat16().float()]) for x in (kr, vr))
    check(got[1:2], attention(q[1, :1].double(), held(kr), held(vr), True, 1, past, 0), torch.float32, max(vr.abs().max().item(), 1))


def test_another_stream(KV8Cache):
    c, k, v = filled(KV8Cache, [700], 2, 64, torch.float32, 14)
    q = torch.randn(1, 1, 2, 64, device='cuda')
    lens = words(700)
    want = c.attend(q, lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.attend(q, lens)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_a_split_call_captured_and_replayed(KV8Cache):
    """A call that needs scratch, captured; replayed at other lengths while eager calls allocate and use theirs."""
    c, k, v = filled(KV8Cache, [9000, 5000], 2, 64, torch.float32, 60)
    other, _, _ = filled(KV8Cache, [7000, 64], 2, 64, torch.float32, 61)
    q = torch.randn(2, 3, 4, 64, device='cuda', generator=torch.Generator(device='cuda').manual_seed(7))
    lens = words(9000, 5000)
    c.attend(q, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.attend(q, lens)
    for a, b in ((9000, 5000), (8999, 1), (64, 4097), (0, 3000)):
        lens.copy_(words(a, b))
        want = c.attend(q, lens).clone()
        g.replay()
        other.attend(q, words(7000, 64))
        torch.cuda.synchronize()
        assert torch.equal(out, want), (a, b)


def test_two_threads_on_two_streams(KV8Cache):
    import threading
    made = [filled(KV8Cache, [5000, 700], 2, 64, torch.bfloat16, 70 + i) for i in range(2)]
    qs = [torch.randn(20, 2, 4, 64, device='cuda').bfloat16() for _ in range(2)]
    lens = words(5000, 700)
    want = [[c.attend(q[:, None], lens).clone() for q in qq] for (c, _, _), qq in zip(made, qs)]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = [made[i][0].attend(q[:, None], lens) for q in qs[i]]
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for g, w in zip(got, want):
        assert len(g) == 20 and all(torch.equal(a, b) for a, b in zip(g, w))


def test_empty_calls(KV8Cache):
    c = KV8Cache(2, 2, 64, 100)
    z = words(0, 0)
    e = torch.zeros(2, 0, 2, 64, device='cuda')
    c.store(e, e, z)
    assert c.attend(e, z).shape == (2, 0, 2, 64)
    assert c.load(z, 0)[0].shape == (2, 2, 0, 64)
    assert (c.attend(torch.ones(2, 3, 2, 64, device='cuda'), z) == 0).all()


def test_refusals(KV8Cache):
    for kw in (dict(head_dim=48), dict(head_dim=0), dict(rows=0), dict(heads=0), dict(capacity=0), dict(dtype=torch.float16),
               dict(device='cpu'), dict(rows=65536)):
        with pytest.raises(ValueError):
            KV8Cache(**{**dict(rows=2, heads=2, head_dim=64, capacity=100), **kw})
    c = KV8Cache(2, 2, 64, 100)
    z, z64 = words(0, 0), torch.zeros(2, dtype=torch.int64, device='cuda')
    x = torch.zeros(2, 5, 2, 64, device='cuda')
    for args in ((x, x, z64), (x, x, z.cpu()), (x, x, z[:1]), (x[:1], x[:1], z), (x, x[:, :4], z), (x, x.bfloat16(), z), (x.half(), x.half(), z),
                 (x[:, :, :1], x[:, :, :1], z), (x[..., :32], x[..., :32], z), (x.cpu(), x.cpu(), z), (x[0], x[0], z), (x, x, z, z64)):
        with pytest.raises(ValueError):
            c.store(*args)
    for args, kw in (((z,), dict(T=129)), ((z,), dict(T=-1)), ((z,), dict(dtype=torch.float16)), ((z64,), {}), ((None,), {})):
        with pytest.raises(ValueError):
            c.load(*args, **kw)
    q, k = torch.zeros(2, 4, 64, device='cuda'), torch.zeros(2, 2, 64, device='cuda')
    for args, kw in (((q[:, :3], k, k, z), {}), ((q, k[:1], k[:1], z), {}), ((q, k, k.bfloat16(), z), {}), ((q, k, k, z64), {}),
                     ((q, k, k, z), dict(past_context=-1)), ((q, k, k, z), dict(starts=z64)), ((q.half(), k, k, z), {}), ((q[:, None], k, k, z), {}),
                     ((q[:, :0], k, k, z), {}), ((q[..., :32], k, k, z), {})):
        with pytest.raises(ValueError):
            c.decode(*args, **kw)
    q = torch.zeros(2, 3, 4, 64, device='cuda')
    for args, kw in (((q[:, :, :3], z), {}), ((q[:1], z), {}), ((q, None), {}), ((q, z), dict(causal=False, past_context=5)),
                     ((q, z), dict(q_lens=z64)), ((q[0], z), {}), ((q.cpu(), z), {})):
        with pytest.raises(ValueError):
            c.attend(*args, **kw)
