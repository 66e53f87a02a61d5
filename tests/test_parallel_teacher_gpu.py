"""A generator that learns from a teacher on two ranks (see tests/dp_teacher.py, which tests/conftest.py starts as a child
process before this session initialises the GPU)."""
import json
import os

import pytest

import conftest

pytestmark = pytest.mark.gpu


def test_two_ranks_with_a_teacher():
    job = conftest.DP_TEACHER
    assert job is not None, "the two ranks were not started (tests/conftest.py starts them for -m gpu sessions)"
    proc, out_path, log_path = job
    try:
        rc = proc.wait(timeout=100)       # (a rank that waits for a missing partner would sit here)
    except Exception:
        proc.kill()
        raise AssertionError("the two ranks did not finish: " + open(log_path).read()[-2000:])
    assert rc == 0 and os.path.exists(out_path), open(log_path).read()[-3000:]
    with open(out_path) as f:
        ranks = json.load(f)
    assert [r["rank"] for r in ranks] == [0, 1]
    for r in ranks:
        # all trainers hold the initial generator then; sums of the ranks' own gradients, in 32 bits
        assert r["grad_mean_err"] <= 1e-6, r
        for what, seen in r["steps"].items():
            assert seen["equal"] and seen["finite"], (what, r)
            assert seen["moved"] > 0, (what, r)
            fails = what != "nothing" and (r["rank"] == 1 or what == "both")
            assert (seen["raised"] is None) != fails and (not fails or "injected" in seen["raised"]), (what, r)
    assert set(ranks[0]["steps"]) == {"nothing", "critic", "draws", "early draws", "distillation", "raw graphs", "both"}
