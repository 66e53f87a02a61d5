"""Which plan a template gets (what a plan holds is made on the GPU; here it is a stand-in that remembers its features)."""
import copy
import pickle

import pytest
import torch

from gan_amd import generator as gen
from gan_amd.data import Data


class Plan:
    def __init__(self, x, K):
        self.features, self.K = x.clone(), K


@pytest.fixture
def made(monkeypatch):
    plans = []

    def build(x, nd, K):
        plans.append(Plan(x, K))
        return plans[-1]
    monkeypatch.setattr(gen.GeneratorPlan, "build", staticmethod(build))
    return plans


def plan_of(G, tpl):
    x = tpl.x if tpl.x.dtype == torch.float32 else tpl.x.float()
    plan = G.plan_for(tpl, x, None)
    assert torch.equal(plan.features, x) and plan.K == G.candidate_k
    return plan


def test_a_plan_is_kept_per_width(made):
    wide, narrow, tpl = gen.AIGGenerator(candidate_k=8), gen.AIGGenerator(candidate_k=4), Data(x=torch.rand(30, 2))
    first = [plan_of(G, tpl) for G in (wide, narrow)]
    for _ in range(3):
        assert [plan_of(G, tpl) for G in (wide, narrow)] == first
    assert len(made) == 2
    tpl.x.add_(1.0)
    assert plan_of(wide, tpl) is not first[0] and plan_of(narrow, tpl) is not first[1]


def test_features_that_take_the_place_of_others(made):
    """Features replaced while one of two generators looks: the other does not take new ones at an old address for the old."""
    wide, narrow, tpl = gen.AIGGenerator(candidate_k=8), gen.AIGGenerator(candidate_k=4), Data(x=torch.rand(5000, 2))
    for k in range(20):
        plan_of(wide, tpl), plan_of(narrow, tpl)
        tpl.x = None
        tpl.x = torch.rand(5000, 2)          # (often the address that has just become free)
        plan_of(wide, tpl)
        tpl.x = None
        tpl.x = torch.rand(5000, 2)
        plan_of(narrow, tpl)


def test_features_in_another_type_are_followed(made):
    """Changed in place: what they are converted to may well be made at the same address again."""
    G, tpl = gen.AIGGenerator(candidate_k=8), Data(x=torch.rand(5000, 2, dtype=torch.float64))
    kept = plan_of(G, tpl)
    assert plan_of(G, tpl) is kept
    for _ in range(5):
        tpl.x.add_(1.0)
        plan_of(G, tpl)


def test_clones_do_not_displace_each_others_plans(made):
    wide, narrow, tpl = gen.AIGGenerator(candidate_k=8), gen.AIGGenerator(candidate_k=4), Data(x=torch.rand(30, 2))
    plan_of(wide, tpl), plan_of(narrow, tpl)
    other = tpl.clone()
    kept = [plan_of(G, t) for t in (tpl, other) for G in (wide, narrow)]
    count = len(made)
    for _ in range(3):
        assert [plan_of(G, t) for t in (tpl, other) for G in (wide, narrow)] == kept
    assert len(made) == count == 4


def test_a_plan_with_windows_can_be_copied_and_pickled():
    """What was enqueued is waited for; the copy has nothing to wait for."""
    class Event:
        waited = 0

        def synchronize(self):
            Event.waited += 1

        def __reduce__(self):
            raise TypeError("an event is not copied")
    plan = gen.GeneratorPlan()
    made = object.__new__(gen._Enqueued)
    made.event, made.stream = Event(), 7
    plan.windows, plan.K = (torch.zeros(3), torch.ones(3), made), 8
    tpl = Data(x=torch.rand(4, 2))
    tpl.__dict__["_gen_plan"] = plan
    for other in (copy.deepcopy(tpl), pickle.loads(pickle.dumps(tpl)), copy.copy(tpl)):
        kept = other.__dict__["_gen_plan"].windows[2]
        assert kept is made or kept.event is None
        assert torch.equal(other.__dict__["_gen_plan"].windows[1], torch.ones(3))
    assert Event.waited == 2 and made.event is not None


def test_a_copy_of_a_template_and_features_at_the_originals_address(made):
    """A copied plan names the original's features, which its copy does not keep alive."""
    G = gen.AIGGenerator(candidate_k=8)
    for _ in range(20):
        tpl = Data(x=torch.rand(5000, 2))
        plan_of(G, tpl)
        other = copy.deepcopy(tpl)
        made.clear()                           # (nothing else holds the original and its plan)
        del tpl
        other.x = torch.rand(5000, 2)          # (often the address that has just become free)
        plan_of(G, other)
