"""Hooks around the optimizer's ``load_state_dict``, and what it leaves of the dicts it is given."""
import copy
import io
import pickle

import pytest
import torch

from adamw_on_cpu import AdamW, make_params, take_steps  # noqa: F401


def test_hooks_see_the_state(AdamW):
    """A pre hook may replace the dict or change its state, a post hook finds the state in place; all of it in the types it had."""
    p, q = make_params(), make_params()
    opt = AdamW(p, lr=0.25)
    take_steps(p, opt, 3)
    saved = copy.deepcopy(opt.state_dict())
    kept = copy.deepcopy(saved)
    other = AdamW(q)
    seen = []

    def pre(o, d):
        seen.append(len(d["state"]))
        state = {k: dict(s, exp_avg=torch.full_like(s["exp_avg"], 0.5)) for k, s in d["state"].items()}
        return dict(d, state=state)

    other.register_load_state_dict_pre_hook(pre)
    other.register_load_state_dict_post_hook(lambda o: seen.append([float(o.state[x]["exp_avg"].sum()) for x in q]))
    other.load_state_dict(saved)
    assert seen == [3, [0.5 * x.numel() for x in q]]
    for k, s in kept["state"].items():
        assert s.keys() == saved["state"][k].keys() and all(torch.equal(s[n], saved["state"][k][n]) for n in s)
    assert all(torch.equal(other.state[x]["exp_avg_sq"], kept["state"][i]["exp_avg_sq"]) for i, x in enumerate(q))
    assert len(other._optimizer_load_state_dict_pre_hooks) == 1             # none of its own is left behind


def test_refused_dicts_change_nothing(AdamW):
    p = make_params()
    opt = AdamW(p, lr=0.25)
    take_steps(p, opt, 2)
    before = copy.deepcopy(opt.state_dict())
    for bad in (torch.optim.AdamW(p, amsgrad=True).state_dict(), torch.optim.AdamW(p[:2]).state_dict()):
        with pytest.raises((RuntimeError, ValueError)):
            opt.load_state_dict(bad)
        now = opt.state_dict()
        assert now["param_groups"] == before["param_groups"] and len(opt._optimizer_load_state_dict_pre_hooks) == 0
        assert all(torch.equal(now["state"][k][n], s[n]) for k, s in before["state"].items() for n in s)


def test_moments_keep_their_type_over_bf16_parameters(AdamW):
    """Also through a file, and with keys of torch's that this class has no use for."""
    p = [torch.nn.Parameter(torch.randn(300).bfloat16())]
    moments = {"exp_avg": torch.randn(300), "exp_avg_sq": torch.rand(300)}
    saved = AdamW(p).state_dict()
    saved["state"] = {0: dict(moments, step=torch.tensor(3.0))}
    file = io.BytesIO()
    torch.save(saved, file)
    file.seek(0)
    opt = AdamW(p)
    opt.load_state_dict(torch.load(file))
    state = opt.state[p[0]]
    assert state.keys() == moments.keys() and all(torch.equal(state[k], moments[k]) for k in moments)


def test_a_copy_loads_and_entries_of_no_parameter_pass(AdamW):
    p = make_params()
    opt = AdamW(p)
    take_steps(p, opt, 2)
    saved = dict(opt.state_dict())
    saved["state"] = dict(saved["state"], note={"text": "kept"})
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        other.load_state_dict(saved)
        q = other.param_groups[0]["params"]
        assert other.state["note"] == {"text": "kept"} and all(torch.equal(other.state[x]["exp_avg"], opt.state[y]["exp_avg"]) for x, y in zip(q, p))
