"""-m gpu: the streaming state of an LMModel with its self-attention cache in 8 bits: what it restores is the cache it was taken from."""
import pytest
import torch

from test_gpu_kv8_lm import conditions, models, sequence

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('wdt', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('t', [40, 64, 65, 130, 192])
def test_a_restored_cache_is_the_same_cache(wdt, t):
    """Codes, scales and newest blocks bit for bit; the logits that follow too."""
    _, b = models(wdt)
    ct, seq = conditions(4, 256), sequence(4, t + 5)
    with b.streaming():
        for i in range(t):
            b(seq[..., i:i + 1], [], ct)
        state = {k: v.clone() for k, v in b.get_streaming_state().items()}
        last = (t - 1) // 64
        caches = b._run['kv8']
        before = [(c.k_codes[:, :, :last].clone(), c.v_codes[:, :, :last].clone(), c.k_scale[:, :, :last].clone(), c.v_scale[:, :, :last].clone(),
                   c.k_tail[:, :, :t - 64 * last].clone(), c.v_tail[:, :, :t - 64 * last].clone()) for c in caches]
        first = b(seq[..., t:], [], ct)
        for c in caches:            # nothing of it left
            for x in (c.k_codes, c.v_codes, c.k_scale, c.v_scale, c.k_tail, c.v_tail):
                x.zero_()
        b.set_streaming_state(state)
        for c, was in zip(caches, before):
            now = (c.k_codes[:, :, :last], c.v_codes[:, :, :last], c.k_scale[:, :, :last], c.v_scale[:, :, :last],
                   c.k_tail[:, :, :t - 64 * last], c.v_tail[:, :, :t - 64 * last])
            for x, y in zip(now, was):
                assert torch.equal(x, y)
        again = b(seq[..., t:], [], ct)
    assert torch.equal(again, first)
