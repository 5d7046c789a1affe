"""The rotary patch (fskernels.hip.hf) where no GPU is needed: host tensors and
other call forms go to the model's own function, and the helpers restore it."""
import types

import pytest
import torch

from fskernels.hip import hf as H


def rotary(q, k, cos, sin, unsqueeze_dim=1):
    return "own", unsqueeze_dim


def test_other_calls_go_to_the_models_function():
    fn = H.hf_rotary(rotary)
    q = torch.zeros(2, 4, 3, 64)
    t = torch.zeros(2, 3, 64)
    assert fn(q, q, t, t) == ("own", 1)
    assert fn(q, q, t, t, 2) == ("own", 2)
    assert fn(q, q, t, t, unsqueeze_dim=2) == ("own", 2)
    assert fn.__name__ == "rotary"
    with pytest.raises(TypeError):
        fn(q, q, t, t, position_ids=None)  # as the function itself says


def test_helpers_install_once_and_restore():
    mod = types.SimpleNamespace(apply_rotary_pos_emb=rotary)
    with H.patched_hf_rotary(mod):
        inner = mod.apply_rotary_pos_emb
        assert inner is not rotary
        assert H.patch_hf_rotary(mod) is inner and mod.apply_rotary_pos_emb is inner
    assert mod.apply_rotary_pos_emb is rotary


def test_default_module_is_qwen3():
    qm = pytest.importorskip("transformers.models.qwen3.modeling_qwen3")
    before = qm.apply_rotary_pos_emb
    with H.patched_hf_rotary():
        assert getattr(qm.apply_rotary_pos_emb, "_fsk_patch", False)
    assert qm.apply_rotary_pos_emb is before
