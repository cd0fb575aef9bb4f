"""-m gpu: the 8-bit cache's attention where the numbers it holds differ in size: what a query does not see, or gives no weight
to, leaves its result alone however large it is.

Every result is held to its own size, sum p |v| over what the query sees (the definition in 64 bits, test_gpu_kv8.held): scores
carry 2^-17 and probabilities 2^-22 (f32 results) or 2^-12 (bf16) of relative error, sums are f32: 2^-15 sum p |v| in f32,
2^-11 sum p |v| + 2^-8 |result| in bf16 (the last its one rounding).  Not seen means no term at all; a token seen with a
probability of e^-100 adds its p |v| < 1e-4 of the rest.
"""
import math

import pytest
import torch

from test_gpu_kv8 import AnyCache, BLK, DT, KV8Cache, held, make, words   # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def expect(q, k, v, lo, hi):
    """q [S, H, hd], k / v [n, H, hd] f64; query i sees [lo[i], hi[i]) -> result, sum p |v|."""
    t = torch.arange(k.shape[0])
    seen = (t[None] >= torch.tensor(lo)[:, None]) & (t[None] < torch.tensor(hi)[:, None])
    s = torch.einsum('shd,thd->hst', q.double(), k) / math.sqrt(q.shape[-1])
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
    return torch.einsum('hst,thd->shd', p, v), torch.einsum('hst,thd->shd', p, v.abs())


def close(got, ref, size, dt):
    bound = 2.0 ** -15 * size if dt == torch.float32 else 2.0 ** -11 * size + 2.0 ** -8 * ref.abs()
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), (err / bound.clamp_min(1e-300)).max().item()


@pytest.mark.parametrize('R', [1e8, 1e12, 3e38])
@pytest.mark.parametrize('what', ['v', 'k'])
@pytest.mark.parametrize('place', ['newest', 'tail before starts', 'block before starts', 'block before the window'])
@pytest.mark.parametrize('dt,S,hd', [('f32', 2, 64), ('f32', 100, 64), ('bf16', 100, 64), ('f32', 70, 128), ('bf16', 20, 16)])
def test_large_and_not_seen(AnyCache, dt, S, hd, place, what, R):
    dt, n, H = DT[dt], 150, 2
    start, past, S = 0, 0, (min(S, 12) if place == 'tail before starts' else S)
    k, v = make(1, n, H, hd, dt, 6)
    x = v if what == 'v' else k
    first = n - S                                    # position of query 0
    if place == 'newest':
        large = range(n - 1, n)                      # every query but the last is before it
    elif place == 'tail before starts':
        start, large = 133, range(129, 133)
    elif place == 'block before starts':
        start, large = 30, range(5, 30)
    else:
        past = 30
        large = range(first - past - 10 if first - past - 10 > 0 else 0, max(first - past, 1))
    sign = torch.where(torch.rand(x[:, large].shape, generator=torch.Generator().manual_seed(1)) < 0.5, -1.0, 1.0)
    x[:, large] = (R * sign).to(dt)
    q = torch.randn(1, S, H, hd, generator=torch.Generator().manual_seed(2)).to(dt)
    c = AnyCache(1, H, hd, 256, dtype=dt)
    c.store(k.cuda(), v.cuda(), words(0))
    got = c.attend(q.cuda(), words(n), past_context=past, starts=words(start))
    kh, vh = held(k[0].float()), held(v[0].float())
    pos = [first + i for i in range(S)]
    lo = [max(start, p - past if past else 0) for p in pos]
    live = [i for i, p in enumerate(pos) if not any(lo[i] <= t <= p for t in large)]
    assert len(live) >= max(S - 1, 1)
    ref, size = expect(q[0, live], kh, vh, [lo[i] for i in live], [pos[i] + 1 for i in live])
    close(got[0, live], ref, size, dt)


@pytest.mark.parametrize('R', [1e9, 1e12, 1e30])
@pytest.mark.parametrize('at', ['tail', 'first block', 'last block'])
@pytest.mark.parametrize('dt,S,hd', [('f32', 1, 64), ('f32', 90, 64), ('bf16', 90, 64), ('f32', 1, 128), ('bf16', 1, 32)])
def test_large_without_weight(AnyCache, dt, S, hd, at, R):
    """A large value whose key puts its score at -100."""
    dt, n, H = DT[dt], 64 * 5 + 40, 1
    k, v = make(1, n, H, hd, dt, 8)
    t = {'tail': n - 3, 'first block': 10, 'last block': 64 * 4 + 5}[at]
    q = torch.randn(1, S, H, hd, generator=torch.Generator().manual_seed(3)).to(dt)
    q[..., 0] = 1.0
    k[:, t] = 0
    k[:, t, :, 0] = -100 * math.sqrt(hd)
    v[:, t] = torch.where(v[:, t] < 0, -R, R).to(dt)
    c = AnyCache(1, H, hd, 512, dtype=dt)
    c.store(k.cuda(), v.cuda(), words(0))
    got = c.attend(q.cuda(), words(n), causal=False)
    ref, size = expect(q[0], held(k[0].float()), held(v[0].float()), [0] * S, [n] * S)
    close(got[0], ref, size, dt)


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('n', [100, 700])
def test_decode_with_a_large_value_in_the_tail(KV8Cache, dt, n):
    """The new token itself and one in the newest block, both at a score of -100."""
    dt, hd, H, G = DT[dt], 64, 2, 2
    k, v = make(2, n + 1, H, hd, dt, 9)
    q = torch.randn(2, H * G, hd, generator=torch.Generator().manual_seed(4)).to(dt)
    q[..., 0] = 1.0
    for r, t in ((0, n), (1, n - 2)):
        k[r, t] = 0
        k[r, t, :, 0] = -800.0
        v[r, t] = torch.where(v[r, t] < 0, -1e14, 1e14).to(dt)
    c = KV8Cache(2, H, hd, 1024, dtype=dt)
    c.store(k[:, :n].cuda(), v[:, :n].cuda())
    got = c.decode(q.cuda(), k[:, n].cuda(), v[:, n].cuda(), words(n, n))
    for r in range(2):
        ref, size = expect(q[r][None], held(k[r].float()).repeat_interleave(G, 1), held(v[r].float()).repeat_interleave(G, 1), [0], [n + 1])
        close(got[r][None], ref, size, dt)


@pytest.mark.parametrize('S', [1, 100])
@pytest.mark.parametrize('n', [1, 30, 64, 200, 6000])
def test_values_near_the_largest_number(AnyCache, S, n):
    """3e38 of one sign: the sum of probabilities times values passes what f32 holds, the result does not."""
    k, v = make(1, n, 1, 64, torch.float32, 10)
    k = k * 0.1
    v = 1e38 + 2e38 * torch.rand(v.shape, generator=torch.Generator().manual_seed(5))
    q = torch.randn(1, S, 1, 64, generator=torch.Generator().manual_seed(6))
    c = AnyCache(1, 1, 64, n, dtype=torch.float32)
    c.store(k.cuda(), v.cuda(), words(0))
    got = c.attend(q.cuda(), words(n), causal=False)
    ref, size = expect(q[0], held(k[0]), held(v[0]), [0] * S, [n] * S)
    close(got[0], ref, size, torch.float32)


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('hd', [16, 32, 64, 128])
def test_a_first_token_comes_back_as_it_is(KV8Cache, dt, hd):
    """One token, probability 1."""
    dt = DT[dt]
    v = (torch.randn(3, 2, hd, generator=torch.Generator().manual_seed(7)) * torch.tensor([1.0, 1e-12, 1e20])[:, None, None]).to(dt).cuda()
    k, q = (torch.randn(3, 2, hd, generator=torch.Generator().manual_seed(8)).to(dt).cuda() for _ in range(2))
    got = KV8Cache(3, 2, hd, 100, dtype=dt).decode(q, k, v, words(0, 0, 0))
    assert torch.equal(got, v)


@pytest.mark.parametrize('R', [2.0 ** 8, 2.0 ** 16, 2.0 ** 40])
@pytest.mark.parametrize('S', [1, 90])
def test_one_large_feature(AnyCache, S, R):
    """A value whose one feature is large and seen: the other features of the result keep their own precision."""
    n, hd = 64 * 4 + 30, 64
    k, v = make(1, n, 1, hd, torch.float32, 11)
    for t in (70, n - 4):
        v[:, t, :, 3] = R
    q = torch.randn(1, S, 1, hd, generator=torch.Generator().manual_seed(9))
    c = AnyCache(1, 1, hd, 512, dtype=torch.float32)
    c.store(k.cuda(), v.cuda(), words(0))
    got = c.attend(q.cuda(), words(n), causal=False)
    ref, size = expect(q[0], held(k[0]), held(v[0]), [0] * S, [n] * S)
    close(got[0], ref, size, torch.float32)


@pytest.mark.parametrize('H,past', [(384, 0), (200, 90)])
def test_bf16_results_to_their_own_size(KV8Cache, H, past):
    """Prompts on a full grid (two column tiles per wave, and one): tight enough that a token left out would show."""
    S, n, hd = 70, 333, 64
    k, v = make(1, n, H, hd, torch.bfloat16, 41)
    q = torch.randn(1, S, H, hd, generator=torch.Generator().manual_seed(42)).bfloat16()
    c = KV8Cache(2, H, hd, n)
    c.store(torch.cat([k, k]).cuda(), torch.cat([v, v]).cuda())
    got = c.attend(torch.cat([q, q]).cuda(), words(n, n), past_context=past)
    hi = [n - S + i + 1 for i in range(S)]
    lo = [max(0, h - 1 - past) if past else 0 for h in hi]
    kh, vh = held(k[0].float()), held(v[0].float())
    ref, size = expect(q[0], kh, vh, lo, hi)
    close(got[0], ref, size, torch.bfloat16)
    close(got[1], ref, size, torch.bfloat16)
    # the bound is one: without one of the tokens most results leave it
    s = torch.einsum('shd,thd->hst', q[0].double(), kh) / math.sqrt(hd)
    t = torch.arange(n)[None]
    seen = (t >= torch.tensor(lo)[:, None]) & (t < torch.tensor(hi)[:, None]) & (t != 250)
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    off = (torch.einsum('hst,thd->shd', p, vh) - ref).abs() > 2.0 ** -11 * size + 2.0 ** -8 * ref.abs()
    assert off.double().mean() > 0.5


@pytest.mark.parametrize('S', [1, 90])
@pytest.mark.parametrize('sizes', [[1e30, 1e-8, 1e30, 1e-30, 1.0], [1e-30, 1e30, 1e-30, 1e30, 1e-30], [1e5, 1.0, 1e-5, 1e5, 1.0], [1e-20, 1.0, 1e20, 1.0, 1e-20]])
@pytest.mark.parametrize('dt', ['f32', 'bf16'])
def test_blocks_of_other_sizes_keep_their_weight(AnyCache, dt, S, sizes):
    """Blocks whose values are far apart in size, equal in weight: the small ones add next to nothing to the result and their whole
    share to the sum that divides it."""
    dt, n, hd = DT[dt], 64 * 4 + 20, 64
    k, v = make(1, n, 1, hd, dt, 12)
    for b, size in enumerate(sizes):
        v[:, b * BLK:(b + 1) * BLK] *= size
    q = torch.randn(1, S, 1, hd, generator=torch.Generator().manual_seed(10)).to(dt)
    c = AnyCache(1, 1, hd, 512, dtype=dt)
    c.store(k.cuda(), v.cuda(), words(0))
    for starts in (0, 64, 128):
        got = c.attend(q.cuda(), words(n), causal=False, starts=words(starts))
        ref, size = expect(q[0], held(k[0].float()), held(v[0].float()), [starts] * S, [n] * S)
        close(got[0], ref, size, dt)


@pytest.mark.parametrize('dt,hd', [('f32', 64), ('bf16', 64), ('f32', 128), ('f32', 32)])
def test_large_and_not_finite_together(AnyCache, dt, hd):
    """The three newest tokens: a key of 1e10, a value of 1e12, a NaN and an infinity; the queries before them see none of it, those
    that see the NaN give NaN, and an infinite value stays in its feature."""
    dt, n, S, H = DT[dt], 150, 40, 2
    k, v = make(1, n, H, hd, dt, 13)
    k[:, 146, :, 1] = 1e10
    v[:, 147] = 1e12
    v[:, 148, :, 5] = math.inf
    k[:, 149] = math.nan
    q = torch.randn(1, S, H, hd, generator=torch.Generator().manual_seed(11)).to(dt)
    q[..., 1] = -q[..., 1].abs()                     # the large key has no weight
    c = AnyCache(1, H, hd, 256, dtype=dt)
    c.store(k.cuda(), v.cuda(), words(0))
    got = c.attend(q.cuda(), words(n)).cpu()
    v[:, 148, :, 5] = 0
    kh, vh = held(k[0].float()), held(v[0].float())
    kh[149] = 0
    hi = [n - S + i + 1 for i in range(S)]
    ref, size = expect(q[0], kh, vh, [0] * S, hi)
    assert got[0, S - 1].isnan().all() and (got[0, S - 2, :, 5] == math.inf).all()
    got[0, S - 2, :, 5] = ref[S - 2, :, 5].to(dt)
    close(got[0, :S - 1], ref[:S - 1], size[:S - 1], dt)


@pytest.mark.parametrize('R', [1e8, 1e20, 3e38])
@pytest.mark.parametrize('dt,hd', [('f32', 64), ('bf16', 64), ('bf16', 128)])
def test_large_and_later_in_a_block(AnyCache, dt, hd, R):
    """Queries in the middle of the second block, whose last tokens, which they do not see, set its scales."""
    dt, n, S, H = DT[dt], 300, 230, 1
    k, v = make(1, n, H, hd, dt, 14)
    v[:, 120:124] = torch.where(v[:, 120:124] < 0, -R, R).to(dt)
    k[:, 124:126] = torch.where(k[:, 124:126] < 0, -R, R).to(dt)
    q = torch.randn(1, S, H, hd, generator=torch.Generator().manual_seed(12)).to(dt)
    c = AnyCache(1, H, hd, 512, dtype=dt)
    c.store(k.cuda(), v.cuda(), words(0))
    got = c.attend(q.cuda(), words(n))
    ref, size = expect(q[0, :50], held(k[0].float()), held(v[0].float()), [0] * 50, [71 + i for i in range(50)])
    close(got[0, :50], ref, size, dt)
