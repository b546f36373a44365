"""What the steps over a cache refuse before anything runs: sizes that they would only
find wrong once the cache had grown."""
from types import SimpleNamespace

import pytest


def _config():
    return SimpleNamespace(num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                           rope_theta=10000.0, rope_scaling=None, hidden_size=256, intermediate_size=512, vocab_size=100,
                           rms_norm_eps=1e-5)


def _cache(capacity=100):
    torch = pytest.importorskip("torch")
    return SimpleNamespace(layers=2, batch=1, kv_heads=2, head_dim=64, capacity=capacity, dtype=torch.float16,
                           device=torch.device("cpu"), weight=torch.zeros(1))


@pytest.mark.parametrize("options,match", [
    (dict(budget=0), "budget"),
    (dict(budget=-5), "budget"),
    (dict(budget=101), "budget"),
    (dict(budget=100), "budget"),                       # no room for the next token
    (dict(budget=16), "positions"),                     # less than the default 4 + 32
    (dict(budget=50, sinks=-1), "positions"),
    (dict(budget=50, recent=-1), "positions"),
    (dict(budget=50, sinks=20, recent=31), "positions"),
])
def test_budgets(pkg, options, match):
    with pytest.raises(ValueError, match=match):
        pkg.CachedAttention(_config(), _cache(), **options)


def test_good_budgets(pkg):
    for options in (dict(), dict(budget=99), dict(budget=36), dict(budget=50, sinks=20, recent=30),
                    dict(budget=1, sinks=0, recent=0)):
        pkg.CachedAttention(_config(), _cache(), **options)


def test_prompt_longer_than_the_cache(pkg):
    """Refused before its buffers are made: the last rows would not see their own keys."""
    from swiftltx_amd.prefill import PrefillStep
    torch = pytest.importorskip("torch")
    weights = SimpleNamespace(config=_config(), layers=[], embed_tokens=SimpleNamespace(weight=torch.zeros(1)))
    for n in (101, 5000):
        with pytest.raises(ValueError, match="capacity"):
            PrefillStep(weights, n, cache=_cache())
