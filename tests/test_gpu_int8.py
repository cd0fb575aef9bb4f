"""-m gpu: the int8 projection (modules.int8_linear.Int8Linear) against its definition in 64 bits.

Tolerances, fixed before the first run (u = 2^-24, one f32 rounding): the codes follow the format's 32-bit rule, computed here
the same way, and the integer sum is exact, so y before the activation differs by its conversion to f32, the scales' two
roundings and their product, one multiply-add and the residual's sum: <= 6 u (|acc sa sw| + |bias| + |residual|); GELU's slope is
below 1.13 and its erf carries 4 u (f32 results) or 4.3e-7 absolute (bf16 results); one rounding to the output type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {'f32': torch.float32, 'bf16': torch.bfloat16}
U = 2.0 ** -24


@pytest.fixture(scope='module')
def Int8Linear():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from audiocraft_amd.modules.int8_linear import Int8Linear
    return Int8Linear


def rows8(x):
    """f32 rows -> (codes f64, scales f64) by the format's rule."""
    amax = x.abs().amax(-1, keepdim=True)
    live = amax >= 2.0 ** -120
    inv = torch.where(live, torch.full_like(amax, 127.0) / amax, torch.zeros_like(amax))
    return torch.round(x * inv).double(), torch.where(live, amax / torch.tensor(127.0), torch.zeros_like(amax)).double()


def reference(x, w, bias, act, residual):
    a, sa = rows8(x.float())
    b, sb = rows8(w.float())
    lin = (a @ b.t()) * sa * sb.t()
    size = lin.abs()
    if bias is not None:
        lin, size = lin + bias.double(), size + bias.double().abs()
    err = 6 * U * size
    y = 0.5 * lin * (1 + torch.erf(lin / math.sqrt(2))) if act == 'gelu' else lin
    if act == 'gelu':
        err = 1.13 * err + 8 * U * lin.abs() + (4.3e-7 if x.dtype == torch.bfloat16 else 0)
    if residual is not None:
        y = y + residual.double()
        err = err + 2 * U * (y.abs() + residual.double().abs())
    return y, err + torch.finfo(x.dtype).eps / 2 * (y.abs() + err)


def check(layer, x, w, bias, act, residual=None):
    got = layer(x.cuda(), None if residual is None else residual.cuda())
    assert got.dtype == x.dtype and got.shape == x.shape[:-1] + (w.shape[0],)
    y, err = reference(x.reshape(-1, x.shape[-1]), w, bias, act, None if residual is None else residual.reshape(-1, w.shape[0]))
    d = (got.cpu().double().reshape(y.shape) - y).abs()
    assert (d <= err).all(), (d - err).max().item()
    return got


def make(M, N, K, dt, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g) * (0.1 + 3 * torch.rand(M, 1, generator=g))).to(dt)
    return x, torch.randn(N, K, generator=g) / math.sqrt(K), torch.randn(N, generator=g)


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('act', ['none', 'gelu'])
@pytest.mark.parametrize('M,N,K', [(1, 1, 1), (1, 16, 64), (1, 1537, 1000), (3, 33, 65), (16, 64, 4096), (17, 100, 63), (33, 48, 200),
                                   (64, 17, 129), (65, 31, 64), (130, 129, 192), (257, 260, 127), (1000, 515, 320),
                                   (4100, 2052, 96)])
def test_linear(Int8Linear, dt, act, M, N, K):
    x, w, bias = make(M, N, K, DT[dt], M + N + K)
    check(Int8Linear(w.cuda(), bias.cuda(), act), x, w, bias, act)


@pytest.mark.parametrize('M,N,K', [(600, 20, 2500), (2049, 18, 2112), (520, 33, 8200), (2060, 17, 9000), (4100, 70, 2050)])
def test_long_rows(Int8Linear, M, N, K):
    """Rows longer than a wave or a workgroup keeps in registers, either way of quantising them."""
    x, w, bias = make(M, N, K, torch.float32, 6)
    check(Int8Linear(w.cuda(), bias.cuda()), x, w, bias, 'none')


def test_results_past_32_bit_offsets(Int8Linear):
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    x, w, bias = make(66000, 33000, 64, torch.bfloat16, 7)
    got = Int8Linear(w.cuda(), bias.cuda())(x.cuda())
    for r in (0, 32600, 65200, 65999):
        y, err = reference(x[r:r + 1], w, bias, 'none', None)
        assert ((got[r].cpu().double() - y[0]).abs() <= err[0]).all(), r


@pytest.mark.parametrize('M', [2, 20, 100])
@pytest.mark.parametrize('N', [96, 95])
def test_residual_no_bias_and_leading_dimensions(Int8Linear, M, N):
    x, w, _ = make(3 * M, N, 256, torch.float32, M)
    res = torch.randn(3, M, N, generator=torch.Generator().manual_seed(1))
    check(Int8Linear(w.cuda()), x.view(3, M, 256), w, None, 'none', res)


@pytest.mark.parametrize('M', [5, 90])
def test_strides(Int8Linear, M):
    x, w, bias = make(M, 64, 130, torch.bfloat16, 2)
    layer = Int8Linear(w.cuda(), bias.cuda())
    want = check(layer, x, w, bias, 'none')
    buf = torch.zeros(M, 301, device='cuda', dtype=torch.bfloat16)
    buf[:, 1:131] = x.cuda()
    assert torch.equal(layer(buf[:, 1:131]), want)                       # odd pitch and offset
    assert torch.equal(layer(x.cuda().t().contiguous().t()), want)       # columns contiguous
    assert torch.equal(layer(x[:1].cuda().expand(M, 130)), want[:1].expand(M, 64))
    wt = torch.zeros(64, 200, device='cuda')
    wt[:, 3:133] = w.cuda()
    assert torch.equal(Int8Linear(wt[:, 3:133], bias.cuda())(x.cuda()), want)


@pytest.mark.parametrize('M', [4, 80])
def test_special_rows(Int8Linear, M):
    """Zero rows and channels, tiny and huge ones; a NaN or an infinity stays in its row (column)."""
    x, w, bias = make(M, 40, 100, torch.float32, 3)
    x[0] = 0
    x[1] *= 1e30
    x[2] *= 1e-33
    w[3] = 0
    w[4] *= 1e-30
    y = check(Int8Linear(w.cuda(), bias.cuda()), x, w, bias, 'none')
    bad, wbad = x.clone(), w.clone()
    bad[3, 7], wbad[5, 9], wbad[6, 2] = math.nan, math.inf, math.nan
    got = Int8Linear(wbad.cuda(), bias.cuda())(bad.cuda())
    keep_r = [i for i in range(M) if i != 3]
    keep_c = [i for i in range(40) if i not in (5, 6)]
    assert got[3].isnan().all() and got[:, 5:7].isnan().all()
    assert torch.equal(got[keep_r][:, keep_c], y[keep_r][:, keep_c])
    bad[3, 7] = -math.inf
    assert Int8Linear(w.cuda())(bad.cuda())[3].isnan().all()


def test_largest_sum(Int8Linear):
    """Every code +-127 over the longest K: the integer sum stays in 32 bits."""
    K = 131072
    x, w = torch.ones(2, K), torch.ones(20, K)
    x[1] = -1
    got = Int8Linear(w.cuda())(x.cuda()).cpu()
    want = torch.tensor([[1.0], [-1.0]]).expand(2, 20) * K
    assert ((got - want).abs() <= 6 * U * K).all()


def test_same_rows_whatever_the_batch(Int8Linear):
    """A token's result does not depend on how many others there are, nor on the form that serves them."""
    x, w, bias = make(300, 70, 333, torch.bfloat16, 4)
    layer = Int8Linear(w.cuda(), bias.cuda())
    whole = layer(x.cuda())
    for n in (1, 16, 40, 64, 65):
        assert torch.equal(layer(x[:n].cuda()), whole[:n])


def test_captured_and_replayed(Int8Linear):
    x, w, bias = make(16, 128, 256, torch.float32, 5)
    layer = Int8Linear(w.cuda(), bias.cuda(), 'gelu')
    buf = x.cuda()
    layer(buf)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer(buf)
    for k in range(4):
        buf.copy_(x * (k + 1) + k)
        g.replay()
        other = layer(torch.randn(100, 256, device='cuda'))
        torch.cuda.synchronize()
        assert torch.equal(out, layer(buf)) and other.shape == (100, 128)


def test_empty_and_from_linear(Int8Linear):
    lin = torch.nn.Linear(50, 30).cuda()
    layer = Int8Linear.from_linear(lin)
    assert layer(torch.zeros(0, 50, device='cuda')).shape == (0, 30)
    assert layer(torch.zeros(2, 0, 50, device='cuda')).shape == (2, 0, 30)
    x = torch.randn(7, 50)
    check(layer, x, lin.weight.detach().cpu(), lin.bias.detach().cpu(), 'none')


def test_repeated_weight_rows(Int8Linear):
    """A weight whose rows are one row in memory."""
    w = torch.randn(1, 64).expand(20, 64)
    layer = Int8Linear(w.cuda()[:1].expand(20, 64))
    check(layer, torch.randn(5, 64), w, None, 'none')


def test_refusals(Int8Linear):
    w = torch.randn(8, 16, device='cuda')
    for bad in (w.cpu(), w[0], w.half(), w[:0], w[:, :0]):
        with pytest.raises(ValueError):
            Int8Linear(bad)
    with pytest.raises(ValueError):
        Int8Linear(w, torch.zeros(9, device='cuda'))
    with pytest.raises(ValueError):
        Int8Linear(w, activation='relu')
    layer = Int8Linear(w)
    x = torch.zeros(2, 16, device='cuda')
    for bad in (x[:, :15], x.cpu(), x.half(), x.double()):
        with pytest.raises(ValueError):
            layer(bad)
    for bad in (torch.zeros(2, 7, device='cuda'), torch.zeros(2, 8, device='cuda', dtype=torch.bfloat16), torch.zeros(2, 8)):
        with pytest.raises(ValueError):
            layer(x, residual=bad)
