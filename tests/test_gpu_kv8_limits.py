"""-m gpu: the largest calls of the 8-bit operators: refused with a ValueError before anything is launched, or served."""
import pytest
import torch

from test_gpu_int8 import Int8Linear   # noqa: F401  (fixture)
from test_gpu_kv8 import KV8Cache, filled, words   # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def test_calls_past_the_limits(KV8Cache, Int8Linear):   # noqa: F811
    c = KV8Cache(2, 1, 16, 64)
    lens, row = words(1, 1), torch.zeros(16, device='cuda', dtype=torch.bfloat16)
    for S, Hq in (((1 << 20) + 1, 1), (1 << 18, 9), (1, 65536)):
        with pytest.raises(ValueError):
            c.attend(row.expand(2, S, Hq, 16), lens)
    with pytest.raises(ValueError):
        c.decode(torch.zeros(16, device='cuda').expand(2, 65536, 16), torch.zeros(2, 1, 16, device='cuda'), torch.zeros(2, 1, 16, device='cuda'), lens)
    layer = Int8Linear(torch.ones(1, 1, device='cuda'))
    with pytest.raises(ValueError):
        layer(torch.zeros(1, 1, device='cuda', dtype=torch.bfloat16).expand((1 << 30) + 1, 1))
    with pytest.raises(ValueError):
        Int8Linear(torch.zeros(1, 1, device='cuda').expand((1 << 25) + 1, 1))


def test_queries_far_apart_in_memory(KV8Cache):   # noqa: F811
    """Rows of queries 2^31 elements apart."""
    if torch.cuda.mem_get_info()[0] < 10 << 30:
        pytest.skip("needs 10 GB")
    c, _, _ = filled(KV8Cache, [100, 90], 2, 64, torch.bfloat16, 1)
    lens = words(100, 90)
    buf = torch.zeros((1 << 31) + 4096, device='cuda', dtype=torch.bfloat16)
    q = buf.as_strided((2, 1, 4, 64), (1 << 31, 256, 64, 1))
    q.copy_(torch.randn(2, 1, 4, 64, generator=torch.Generator().manual_seed(1)))
    near = q.contiguous()
    assert torch.equal(c.attend(q, lens), c.attend(near, lens))
    k = torch.randn(2, 2, 64, device='cuda').bfloat16()
    assert torch.equal(c.decode(q[:, 0], k, k, lens), c.decode(near[:, 0], k, k, lens))
    wide = buf.as_strided((2, 3, 4, 64), (1 << 31, 256, 64, 1))
    assert torch.equal(c.attend(wide, lens), c.attend(wide.contiguous(), lens))
