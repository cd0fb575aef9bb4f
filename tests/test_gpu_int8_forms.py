"""-m gpu: every form of the int8 projection (fused, streamed, tiles of 128 x 128 and of 256 x 256) gives a token the same result.

Tolerances against the 64-bit definition: test_gpu_int8.reference.  Between the forms: none, the integer sums are exact and what
follows them is the same arithmetic.
"""
import math

import pytest
import torch

from test_gpu_int8 import DT, Int8Linear, make, reference   # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu

# a size for each form at N = 1026 (no multiple of 4), K = 1030 (17 fragments, the last partial): 1 and 16 rows fused, 17 .. 200 streamed,
# from 1409 rows (11 x 9 tiles) 128 x 128 tiles; at N = 4095 4093 rows fill the chip with 256 x 256 tiles
SIZES = [(1026, [1, 16, 17, 40, 64, 200, 1409]), (4095, [1, 16, 33, 130, 4093])]


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('act', ['none', 'gelu'])
@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('N,rows', SIZES)
def test_the_form_does_not_matter(Int8Linear, N, rows, act, residual, dt):
    K, M = 1030, max(rows)
    x, w, bias = make(M, N, K, DT[dt], N)
    w *= 3.0                       # (GELU's whole range)
    res = torch.randn(M, N, generator=torch.Generator().manual_seed(1)) if residual else None
    layer = Int8Linear(w.cuda(), bias.cuda(), act)
    xd, rd = x.cuda(), res.cuda() if residual else None
    whole = layer(xd, rd)
    at = torch.randperm(M, generator=torch.Generator().manual_seed(2))[:150]
    y, err = reference(x[at], w, bias, act, res[at] if residual else None)
    d = (whole[at.cuda()].cpu().double() - y).abs()
    assert (d <= err).all(), (d - err).max().item()
    for n in rows[:-1]:
        assert torch.equal(layer(xd[:n], rd[:n] if residual else None), whole[:n]), n
        assert torch.equal(layer(xd[M - n:], rd[M - n:] if residual else None), whole[M - n:]), n


@pytest.mark.parametrize('N,M', [(1026, 1409), (4095, 4093)])
def test_special_rows_in_the_tiled_forms(Int8Linear, N, M):
    """Zero, tiny and huge rows and channels; a NaN or an infinity stays in its row (column); rows of an odd pitch."""
    K = 1030
    x, w, bias = make(M, N, K, torch.bfloat16, 3)
    x[0], w[3] = 0, 0
    x[M // 2] *= 2.0 ** 90
    x[M - 1] *= 2.0 ** -100
    w[N - 1] *= 2.0 ** -90
    layer = Int8Linear(w.cuda(), bias.cuda())
    buf = torch.zeros(M, K + 3, dtype=torch.bfloat16, device='cuda')[:, 1:K + 1]
    buf.copy_(x)
    whole = layer(buf)
    at = torch.tensor([0, 1, 17, M // 2, M - 2, M - 1])
    y, err = reference(x[at], w, bias, 'none', None)
    assert ((whole[at.cuda()].cpu().double() - y).abs() <= err).all()
    bad, wbad = x.clone(), w.clone()
    bad[200, 7], bad[M - 3, K - 1], wbad[5, 9], wbad[N - 2, K - 1] = math.nan, -math.inf, math.inf, math.nan
    got = Int8Linear(wbad.cuda(), bias.cuda())(bad.cuda())
    keep_r, keep_c = torch.ones(M, dtype=torch.bool, device='cuda'), torch.ones(N, dtype=torch.bool, device='cuda')
    keep_r[[200, M - 3]], keep_c[[5, N - 2]] = False, False
    assert got[~keep_r].isnan().all() and got[:, ~keep_c].isnan().all()
    assert torch.equal(got[keep_r][:, keep_c], whole[keep_r][:, keep_c])


@pytest.mark.parametrize('M', [1, 100, 1500])
def test_gelu_in_bfloat16_to_its_own_size(Int8Linear, M):
    """Results of GELU far out on the negative side, to a bf16 rounding of themselves (relative, not to 1): x from -9 to 9 through a
    weight of one column, whose codes are all 127.

    y carries 6 roundings of 2^-24, which far out |d log gelu / dx| <= |x| + 1 multiplies; erfc by its polynomial 2^-18."""
    N = 1200
    w = torch.linspace(-9.0, 9.0, N).view(N, 1)
    x = torch.ones(M, 1, dtype=torch.bfloat16)
    got = Int8Linear(w.cuda(), activation='gelu')(x.cuda()).cpu().double()
    lin = w.double().view(1, N)
    want = 0.5 * lin * torch.special.erfc(-lin / math.sqrt(2))
    bound = (2.0 ** -8 + 2.0 ** -18 + 6 * 2.0 ** -24 * (lin.abs() + 1) * lin.abs().clamp_min(1)) * want.abs()
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / want.abs().clamp_min(1e-300)).max().item()


def test_the_layer_keeps_its_own_bias(Int8Linear):
    """Built once: neither the weight nor the bias follows what the caller does to its tensors later."""
    x, w, bias = make(4, 32, 64, torch.float32, 9)
    wd, bd = w.cuda(), bias.cuda()
    layer = Int8Linear(wd, bd)
    want = layer(x.cuda())
    wd.zero_()
    bd.zero_()
    assert torch.equal(layer(x.cuda()), want)


def test_very_many_rows(Int8Linear):
    """2^26 rows and some: more work items than one launch takes."""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB")
    M = (1 << 26) + 5
    w = torch.tensor([[1.5], [-0.5], [3.0]])
    layer = Int8Linear(w.cuda())
    x = torch.zeros(M, 1, dtype=torch.bfloat16, device='cuda')
    for at in (0, 1 << 25, (1 << 26) - 1, M - 5, M - 1):
        x[at] = 2.0 + at % 7
    got = layer(x)
    for at in (0, 1 << 25, (1 << 26) - 1, M - 5, M - 1):
        assert ((got[at].cpu().double() - x[at].cpu().double() * w[:, 0].double()).abs() <= 2.0 ** -7 * (2.0 + at % 7) * 3).all()
        x[at] = 0
    assert (layer(x) == 0).all()
