"""Observation tokens behind the end of the position table never reach the device."""
import pytest
import torch

from neko_amd.policy.gato_policy import build_layout, check_positions


@pytest.mark.parametrize("n", [1, 63, 64])
def test_inside(n):
    check_positions(build_layout([{"text": list(range(n))}, {"text": [1]}], True, 64, False).desc, 64)


@pytest.mark.parametrize("batch", [[{"text": list(range(65))}], [{"text": [1, 2]}, {"text": list(range(200))}],
                                   [{"continuous_obs": torch.zeros(2, 70), "continuous_actions": torch.zeros(2, 1)}]], ids=["65", "200", "obs"])
def test_behind(batch):
    pb = build_layout(batch, True, 64, False)
    with pytest.raises(ValueError, match="position table"):
        check_positions(pb.desc, 64)
    check_positions(build_layout(batch, False, 64, False).desc, 64)          # without local positions there is nothing to leave


@pytest.mark.gpu
def test_entry_points_refuse(monkeypatch):
    from test_speculative_gpu import _policy, _prompt
    m = _policy(ctx=64)
    with pytest.raises(ValueError, match="position table"):
        m.predict_text(_prompt(65), max_length=1)
    with pytest.raises(ValueError, match="position table"):
        m.forward([_prompt(65)], compute_loss=True)
    assert m.predict_text(_prompt(64), max_length=1)[0].shape[0] == 1
    asked = []
    real = m.tokenize_input_dicts
    monkeypatch.setattr(m, "tokenize_input_dicts", lambda x: asked.append(x) or real(x))
    with pytest.raises(ValueError, match="exceeds context_len"):
        m.predict_response(torch.zeros(1, 3, 32, 32), prompt_tokens=list(range(61)), max_length=1)          # 4 patches + 61
    assert not asked
