"""Sampling of one token, and drafted decoding at temperatures and logits where a softmax in 32 bits has no answer."""
import math

import pytest
import torch

from neko_amd.policy.gato_policy import sample_token


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("temperature", [1e-300, 1e-45, 1e-40, 1e-12, 1e-3])
def test_cold_is_the_largest(temperature):
    """(A softmax of logits / temperature overflows in 32 bits here and gives NaN, which torch.multinomial refuses.)"""
    for seed in range(5):
        x = torch.randn(500, generator=_gen(seed)) * 4
        assert int(sample_token(x, temperature, _gen(9))) == int(x.argmax())
    if temperature < 1e-38:
        with pytest.raises(RuntimeError):
            torch.multinomial(torch.softmax(x / temperature, -1), 1)


def test_rows_that_are_not_all_numbers():
    x = torch.randn(50, generator=_gen(0))
    x[3], x[7] = math.nan, -math.inf
    for seed in range(50):
        assert int(sample_token(x, 5.0, _gen(seed))) not in (3, 7)
    x[11] = x[20] = math.inf
    assert {int(sample_token(x, 1.0, _gen(s))) for s in range(50)} == {11, 20}
    for bad in (math.nan, -math.inf):
        assert 0 <= int(sample_token(torch.full((9,), bad), 1.0, _gen(0))) < 9


def test_distribution_and_stream():
    """Frequencies of N draws within 4 sigma; and at ordinary temperatures the very draws of torch.multinomial."""
    x, N = torch.tensor([0.3, -1.0, 1.2, 0.0, -30.0]), 20000
    p = torch.softmax(x.double() / 0.8, 0)
    g = _gen(1)
    f = torch.bincount(torch.stack([sample_token(x, 0.8, g) for _ in range(N)]), minlength=5).double() / N
    assert bool(((f - p).abs() <= 4 * (p * (1 - p) / N).sqrt() + 1e-12).all())
    a, b = _gen(2), _gen(2)
    for i in range(200):
        y = torch.randn(128, generator=_gen(i)) * 3
        assert int(sample_token(y, 0.9, a)) == int(torch.multinomial(torch.softmax(y / 0.9, -1), 1, generator=b))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_drafted_decoding_at_the_ends(kind):
    """Next to temperature 0 the answer is the greedy one; logits without a number raise before anything is sampled; a draft whose logits hold none costs
    only its proposals; temperatures outside (0, largest float] are refused."""
    from test_speculative_gpu import _policy, _prompt
    m, draft = _policy(seed=0), _policy(seed=5, layers=1)
    m.kv_cache = draft.kv_cache = kind
    want, greedy = m.predict_text_speculative(_prompt(20), draft, max_length=10)
    for temperature in (1e-40, 1e-20):
        _, t = m.predict_text_speculative(_prompt(20), draft, max_length=10, deterministic=False, temperature=temperature)
        assert [int(x) for x in t] == [int(x) for x in greedy]
    for temperature in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            m.predict_text_speculative(_prompt(20), draft, max_length=4, deterministic=False, temperature=temperature)
    with torch.no_grad():
        dict(draft.named_parameters())["predict_token.weight"].fill_(float("nan"))
    draft._flat.ensure_shadow()
    _, t = m.predict_text_speculative(_prompt(20), draft, max_length=10, deterministic=False, temperature=1e-20)
    assert [int(x) for x in t] == [int(x) for x in greedy]
    for deterministic in (True, False):
        with pytest.raises(RuntimeError, match="no number"):
            draft.predict_text_speculative(_prompt(20), m, max_length=4, deterministic=deterministic)
