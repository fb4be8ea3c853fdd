"""The modules around the convolution without a GPU: what casts, moves and switches do to them."""
import copy

import pytest
import torch

from savanna_amd.operators.block import MixerBlock
from savanna_amd.operators.linear_attention import LinearAttention


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(),
                                  lambda m: m.to("cpu", torch.float16), lambda m: m.bfloat16().float()])
@pytest.mark.parametrize("inside", [False, True])
def test_decays_stay_float32(gcg_lib, cast, inside):
    """Whatever a model is cast to, its linear attention keeps the decays it was made with; its parameters are cast."""
    mixer = LinearAttention(128, 4)
    before = mixer.log_decay.clone()
    whole = MixerBlock(128, mixer) if inside else mixer
    want = cast(torch.nn.Linear(1, 1)).weight.dtype
    assert cast(whole) is whole
    assert mixer.log_decay.dtype == torch.float32 and torch.equal(mixer.log_decay, before)
    assert all(p.dtype == want for p in whole.parameters())
    assert dict(whole.named_buffers())["mixer.log_decay" if inside else "log_decay"] is mixer.log_decay
    moved = copy.deepcopy(whole).to("meta", torch.bfloat16)
    assert all(b.is_meta and b.dtype == torch.float32 for b in moved.buffers())


def test_decays_of_a_model_made_in_another_default_type(gcg_lib):
    try:
        for dtype in (torch.bfloat16, torch.float64):
            torch.set_default_dtype(dtype)
            assert LinearAttention(128, 4).log_decay.dtype == torch.float32
    finally:
        torch.set_default_dtype(torch.float32)


@pytest.mark.parametrize("mixers,block", [(False, False), (False, True), (True, False), (True, True)])
def test_a_block_does_not_switch_a_mixers_checkpoint_off(gcg_lib, mixers, block):
    from savanna_amd.operators.hyena import HyenaMixer, HyenaSEOperator

    for mixer in (LinearAttention(128, 4, save_8bit=mixers), HyenaMixer(HyenaSEOperator(128, 8), save_8bit=mixers)):
        layer = MixerBlock(128, mixer, save_8bit=block)
        assert layer.mixer.save_8bit == (mixers or block) and layer.norm.save_8bit == block


def test_mixers_pickled_before_there_was_a_checkpoint(gcg_lib):
    """Such a module lacks the switch and goes on as it did."""
    from savanna_amd.operators.hyena import HyenaMixer, HyenaSEOperator

    mixer = HyenaMixer(HyenaSEOperator(128, 8))
    del mixer.__dict__["save_8bit"]
    assert not mixer._save_8bit()
    mixer.save_8bit = True
    assert mixer._save_8bit()
