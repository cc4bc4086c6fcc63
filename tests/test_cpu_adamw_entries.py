"""Entries of the optimizer's state that were taken away or replaced between steps."""
import collections

import pytest
import torch

from adamw_on_cpu import AdamW, make_params, take_steps, assert_same  # noqa: F401


def test_state_that_was_taken_away_starts_at_zero(AdamW):
    """As with torch's class: clearing the state, or one parameter's, resets the moments."""
    for reset in (lambda o, p: o.state.clear(), lambda o, p: setattr(o, "state", collections.defaultdict(dict)), lambda o, p: [o.state.pop(x) for x in p]):
        p = make_params()
        opt = AdamW(p)
        take_steps(p, opt, 3)
        q = [torch.nn.Parameter(x.detach().clone()) for x in p]
        fresh = AdamW(q)
        fresh.param_groups[0]["step_count"] = 3
        reset(opt, p)
        take_steps(p, opt, 2, seed=7)
        take_steps(q, fresh, 2, seed=7)
        assert_same(p, q)
    p, q = make_params(), make_params()
    opt, other = AdamW(p), AdamW(q)
    take_steps(p, opt, 3)
    take_steps(q, other, 3)
    del opt.state[p[1]]
    for k in ("exp_avg", "exp_avg_sq"):
        other.state[q[1]][k].zero_()                                        # in place it has always counted
    take_steps(p, opt, 2, seed=7)
    take_steps(q, other, 2, seed=7)
    assert_same(p, q)


def test_entries_that_were_replaced_count(AdamW):
    p, q = make_params(), make_params()
    opt, other = AdamW(p), AdamW(q)
    take_steps(p, opt, 3)
    take_steps(q, other, 3)
    opt.state[p[2]]["exp_avg"] = torch.full((300,), 0.25)
    opt.state[p[0]] = {k: 2 * t for k, t in opt.state[p[0]].items()}
    other.state[q[2]]["exp_avg"].fill_(0.25)
    for t in other.state[q[0]].values():
        t.mul_(2)
    take_steps(p, opt, 2, seed=7)
    take_steps(q, other, 2, seed=7)
    assert_same(p, q)


def test_a_parameter_that_changes_its_type_and_back(AdamW):
    """The moments go along: none of an earlier time come back."""
    p, q = make_params(), make_params()
    opt, other = AdamW(p), AdamW(q)
    for params, o in ((p, opt), (q, other)):
        take_steps(params, o, 2)
        for x in params:
            x.data, x.grad = x.data.bfloat16(), None
        take_steps(params, o, 1, seed=3)
        for x in params:
            x.data, x.grad = x.data.float(), None
        o._moments = o._moments if o is opt else {}                         # the other one makes its buffers anew from the state
        take_steps(params, o, 1, seed=4)
    assert_same(p, q)


def test_a_parameter_that_changes_its_shape_is_refused(AdamW):
    p = make_params()
    opt = AdamW(p)
    take_steps(p, opt, 2)
    p[1].data, p[1].grad = torch.randn(4), None
    with pytest.raises(RuntimeError, match="shape"):
        take_steps(p, opt, 1)


def test_other_entries_are_left_alone(AdamW):
    p, q = make_params(), make_params()
    opt, other = AdamW(p), AdamW(q)
    for k in range(3):
        take_steps(p, opt, 1, seed=k)
        take_steps(q, other, 1, seed=k)
        opt.state[p[0]]["note"], opt.state["all"] = k, "text"
    assert opt.state[p[0]]["note"] == 2 and opt.state["all"] == "text"
    assert_same(p, q)


def test_buffers_stay_where_nothing_was_replaced(AdamW):
    p = make_params()
    p[1].data = p[1].data.bfloat16()
    opt = AdamW([{"params": p[:2]}, {"params": p[2:]}])
    take_steps(p, opt, 1)
    where = {k: (m.avg.data_ptr(), m.sq.data_ptr()) for k, m in opt._moments.items()}
    assert len(where) == 3
    take_steps(p, opt, 3)
    assert where == {k: (m.avg.data_ptr(), m.sq.data_ptr()) for k, m in opt._moments.items()}
