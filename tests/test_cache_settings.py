"""Settings of the decode caches that do not go together are refused by one rule (no GPU needed)."""
from types import SimpleNamespace

import pytest
import torch

from neko_amd.policy.gato_policy import GatoPolicy


def _ask(kv_cache="bf16", window=0, sinks=0):
    return GatoPolicy._cache_dtype(SimpleNamespace(kv_cache=kv_cache, decode_window=window, decode_sinks=sinks))


def test_settings_that_go_together():
    assert _ask() == torch.bfloat16 and _ask("int8") == torch.int8 and _ask("e4m3", 16) == torch.float8_e4m3fn and _ask("int8", 16, 4) == torch.int8


@pytest.mark.parametrize("kw,match", [(dict(kv_cache="fp4"), "kv_cache"), (dict(window=16), "decode_window"), (dict(kv_cache="int8", sinks=4), "decode_sinks"), (dict(sinks=4), "decode_sinks"),
                                      (dict(kv_cache="int8", window=-1), "negative"), (dict(kv_cache="int8", window=8, sinks=-1), "negative")], ids=str)
def test_settings_that_do_not(kw, match):
    with pytest.raises(ValueError, match=match):
        _ask(**kw)


@pytest.mark.gpu
def test_settings_are_looked_at_in_every_call():
    """A decoder of an earlier call is at hand: it is not used under settings that it does not have."""
    from test_speculative_gpu import _policy, _prompt
    m = _policy(ctx=64)
    want, _ = m.predict_text(_prompt(20), max_length=4)
    m.decode_window = 16
    for length in (1, 4):
        with pytest.raises(ValueError, match="decode_window"):
            m.predict_text(_prompt(20), max_length=length)
        with pytest.raises(ValueError, match="decode_window"):
            m.predict_text(_prompt(20), max_length=length, deterministic=False)
    m.decode_window, m.decode_sinks, m.kv_cache = 0, 3, "int8"
    with pytest.raises(ValueError, match="decode_sinks"):
        m.predict_text(_prompt(20), max_length=4)
    m.decode_sinks, m.kv_cache = 0, "bf16"
    assert torch.equal(m.predict_text(_prompt(20), max_length=4)[0], want)
