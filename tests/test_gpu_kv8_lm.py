"""-m gpu: LMModel with its self-attention cache in 8 bits (kv_dtype=torch.int8).

Within the newest 64 positions the cache is exact, so f32 models agree with the f32 cache to summation order (gate 1e-4, as every
f32 logits test of this suite); beyond, int8 with a scale per 64 positions and head is held to the gate of the bf16 models, 3e-2.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30)).item()


def models(wdt=torch.float32, dims=(256, 4, 3), **kw):
    """The same weights with the cache in the weights' type and in 8 bits."""
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from audiocraft_amd.models import builders
    dim, heads, layers = dims
    cfg = dict(dim=dim, num_heads=heads, num_layers=layers, n_q=4, card=512, hidden_scale=4, cfg_coef=3.0,
               conditioners={'description': {'kind': 't5', 'embedder': 'synthetic', 'dim': 64, 'length': 6}},
               **{'fuser': {'cross': ['description']}, **kw})
    out = []
    for kv in (None, torch.int8):
        torch.manual_seed(0)
        out.append(builders.get_lm_model(cfg, 'cuda', wdt, kv))
    return out


def conditions(rows, dim, live=None):
    cross = torch.randn(rows, 6, dim, generator=torch.Generator().manual_seed(5))
    cross[live if live is not None else rows:] = 0
    return {'description': (cross.cuda(), torch.ones(rows, 6, dtype=torch.int64).cuda())}


def sequence(rows, S, seed=6):
    return torch.randint(0, 513, (rows, 4, S), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize('dims', [(256, 4, 3), (128, 8, 2), (256, 2, 2), (128, 4, 2)])   # head sizes 64, 16, 128, 32
def test_the_first_64_positions_are_exact(dims):
    a, b = models(dims=dims)
    ct, seq = conditions(6, dims[0]), sequence(6, 64)
    assert rel(b.forward_steps(seq, ct), a.forward_steps(seq, ct)) < 1e-4
    assert 'k' not in b._run and len(b._run['kv8']) == dims[2]


def test_bounded_context():
    a, b = models(past_context=9)
    ct, seq = conditions(4, 256), sequence(4, 60)
    assert rel(b.forward_steps(seq, ct), a.forward_steps(seq, ct)) < 1e-4


@pytest.mark.parametrize('wdt', [torch.float32, torch.bfloat16])
def test_past_the_first_block(wdt, monkeypatch):
    """230 positions; layer 0's keys and values, which no attention precedes, are the quantised ones of the plain cache (whose QKV
    product is kept a launch of its own too: fused with the attention it sums in another order)."""
    from test_gpu_kv8 import held
    a, b = models(wdt)
    monkeypatch.setattr(type(a), 'QKV_ATTN_FUSED', False)
    ct, seq = conditions(6, 256), sequence(6, 230)
    assert rel(b.forward_steps(seq, ct), a.forward_steps(seq, ct)) < 3e-2
    k, v = b._run['kv8'][0].load(torch.full((6,), 230, dtype=torch.int32, device='cuda'), 230)
    for got, plain in ((k, a._run['k'][0]), (v, a._run['v'][0])):
        for r in range(6):
            ref = held(plain[r, :, :230].float().transpose(0, 1).cpu()).transpose(0, 1)
            off = int(((got[r].cpu().double() - ref).abs() > 3 * 2.0 ** -24 * ref.abs()).sum())
            assert off == 0, off


@pytest.mark.parametrize('wdt', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('prefill', ['big', 'chunk'])
def test_generate_with_a_prompt(wdt, prefill, monkeypatch):
    """A 75-step prompt, then generation: captured and eager steps give the same tokens and logits; the logits stay near the plain
    cache's while the tokens agree."""
    monkeypatch.setenv('ACMI_PREFILL', prefill)
    a, b = models(wdt)
    B = 3
    ct = conditions(2 * B, 256, live=B)
    prompt = torch.randint(0, 512, (B, 4, 75), generator=torch.Generator().manual_seed(8))
    kw = dict(num_samples=B, max_gen_len=150, use_sampling=False, condition_tensors=ct, return_logits=True)
    t0, l0 = a.generate(prompt, [], **kw)
    t1, l1 = b.generate(prompt, [], **kw)
    t2, l2 = b.generate(prompt, [], use_graph=False, **kw)
    assert torch.equal(t1, t2) and torch.equal(l1, l2)
    assert rel(l1[:, :, 0], l0[:, :, 0]) < 3e-2        # the first decision: same past


@pytest.mark.parametrize('fuser', ['cross', 'prepend'])
def test_two_step_guidance(fuser):
    """Conditional and unconditional rows of their own condition length; prepended, the shorter stream is padded on the left and its
    first positions are never seen.  Within 64 positions as with the plain cache, beyond captured and eager steps agree."""
    a, b = models(fuser={fuser: ['description']})
    B = 2

    def source(n, seed):
        return {'description': (torch.randn(B, n, 256, generator=torch.Generator().manual_seed(seed)).cuda(), torch.ones(B, n, dtype=torch.int64).cuda())}
    kw = dict(num_samples=B, use_sampling=False, condition_tensors=(source(6, 1), source(2, 2)), return_logits=True)
    (t0, l0), (t1, l1) = (m.generate(None, [], max_gen_len=40, **kw) for m in (a, b))
    assert torch.equal(t0, t1) and rel(l1, l0) < 1e-4
    (t2, l2), (t3, l3) = (b.generate(None, [], max_gen_len=150, use_graph=g, **kw) for g in (True, False))
    assert torch.equal(t2, t3) and torch.equal(l2, l3) and torch.isfinite(l2).all()


def test_streaming_state_goes_out_and_in():
    _, b = models()
    ct, seq = conditions(4, 256), sequence(4, 150)
    full = b(seq, [], ct)
    with b.streaming():
        parts = [b(seq[..., :1], [], ct), b(seq[..., 1:100], [], ct)]
        state = b.get_streaming_state()
        assert state['transformer.layers.0.self_attn.past_keys'].shape == (4, 4, 100, 64)
        first = b(seq[..., 100:], [], ct)
        b.set_streaming_state(state)
        again = b(seq[..., 100:], [], ct)
    assert rel(torch.cat(parts + [first], dim=2), full) < 1e-4
    # the restored cache holds the same codes (scales to an ulp) and the same newest block
    assert rel(again, first) < 1e-4


def test_musicgen_takes_the_option():
    from audiocraft_amd.models import MusicGen
    m = MusicGen.get_random_init('facebook/musicgen-small', kv_dtype=torch.int8)
    assert m.lm.kv_int8 and m.lm.kv_dtype == m.lm.weight_dtype
    m.set_generation_params(duration=2)
    assert m.generate(['one', 'two']).shape[0] == 2


def test_refusals():
    for kw in (dict(positional_embedding='rope'), dict(qk_layer_norm=True)):
        with pytest.raises(NotImplementedError):
            models(**kw)
    with pytest.raises(NotImplementedError):
        models(dims=(64, 8, 1))
