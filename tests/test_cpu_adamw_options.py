"""What the optimizer's constructor was told and what a loaded state dict says."""
import copy
import pickle

import pytest
import torch

from adamw_on_cpu import AdamW, make_params, take_steps  # noqa: F401


def _options(opt):
    return [(g["state_bits"], g["stochastic_rounding"], g["seed"]) for g in opt.param_groups]


def test_a_dict_of_torch_keeps_what_the_constructor_was_told(AdamW):
    p = make_params()
    ref = torch.optim.AdamW([{"params": p[:2]}, {"params": p[2:], "lr": 0.5}], lr=0.25)
    take_steps(p, ref, 3)
    opt = AdamW([{"params": p[:2]}, {"params": p[2:], "seed": 5}], state_bits=8, seed=77, stochastic_rounding=False)
    opt.load_state_dict(ref.state_dict())
    assert _options(opt) == [(8, False, 77), (8, False, 5)]
    assert [g["lr"] for g in opt.param_groups] == [0.25, 0.5] and [g["step_count"] for g in opt.param_groups] == [3, 3]


@pytest.mark.parametrize("bits,others", [(8, 32), (32, 8)])
def test_a_dict_of_the_other_bits_does_not_change_the_form(AdamW, bits, others):
    """Options that the dict has (seed, rounding) come from it as its learning rate does; how the moments are held is the constructor's choice."""
    p = make_params()
    saved = AdamW(p, state_bits=others, seed=9, stochastic_rounding=False, lr=0.125).state_dict()
    opt = AdamW(p, state_bits=bits)
    opt.load_state_dict(saved)
    assert _options(opt) == [(bits, False, 9)] and opt.param_groups[0]["lr"] == 0.125
    assert saved["param_groups"][0]["state_bits"] == others                # the caller's dict is as it was


def test_a_fresh_dict_of_torch_starts_over(AdamW):
    p = make_params()
    opt = AdamW(p)
    take_steps(p, opt, 4)
    opt.load_state_dict(torch.optim.AdamW(p).state_dict())
    assert opt.param_groups[0]["step_count"] == 0 and not opt.state


def test_copies_and_pickles_keep_the_options(AdamW):
    p = make_params()
    opt = AdamW(p, state_bits=8, seed=77, stochastic_rounding=False, max_grad_norm=2.0)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert _options(other) == _options(opt) and other.max_grad_norm == 2.0
