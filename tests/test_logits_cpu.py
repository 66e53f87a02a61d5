"""What the entry points on rows of logits refuse before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch

from gan_amd import _abi
from gan_amd import logits as L

P = C.c_void_p(4096)      # never read: every call below is refused on its sizes


def test_cpu_tensors_are_refused():
    x, u = torch.zeros(2, 4), torch.zeros(2, 1)
    for call in (lambda: L.sample_rows(x, u), lambda: L.top_rows(x, 2), lambda: L.distill_loss(x, L.TopRows(x, x.int(), None), tail=False),
                 lambda: L.class_scores(x, L.ScoreWindows(*[torch.zeros(2, dtype=torch.int32)] * 6))):
        with pytest.raises(_abi.AigAbiError):
            call()


@pytest.mark.parametrize("rows,width,ld,dtype,draws,rc", [(-1, 4, 4, 0, 1, -1), (4, 0, 4, 0, 1, -1), (4, 4, -1, 0, 1, -1), (4, 4, 4, 3, 1, -1),
                                                          (4, 4, 4, 0, 0, -1), (4, 4, 4, 0, 9, -1), (4, 131073, 131073, 0, 1, -4),
                                                          (1 << 22, 1025, 1025, 0, 1, -4), (1 << 26, 4, 4, 0, 1, -4), (0, 4, 4, 0, 1, 0)])
def test_sample_sizes(rows, width, ld, dtype, draws, rc):
    how = _abi.Sampling(temperature=1.0, top_p=1.0)
    assert _abi.lib().aig_sample_rows(rows, width, ld, dtype, P, None, None, C.byref(how), draws, P, P, None) == rc
    assert _abi.lib().aig_sample_rows(4, 4, 4, 0, P, None, None, None, 1, P, P, None) == -1
    assert _abi.lib().aig_sample_rows(4, 4, 4, 0, None, None, None, C.byref(how), 1, P, P, None) == -1


@pytest.mark.parametrize("m,temperature,rc", [(0, 1.0, -1), (257, 1.0, -1), (4, 0.0, -1), (4, -2.0, -1), (4, float("nan"), -1), (4, 1e-7, -1),
                                              (4, float("inf"), -1)])
def test_top_arguments(m, temperature, rc):
    assert _abi.lib().aig_top_rows(4, 8, 8, 0, P, None, m, temperature, P, P, P, None) == rc


def distill(**kw):
    a = _abi.Distill(rows=4, width=8, ld=8, m=2, dtype=0, temperature=1.0, scale=1.0, logits=4096, values=4096, index=4096)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [(dict(rows=-1), -1), (dict(width=0), -1), (dict(m=0), -1), (dict(m=257), -1), (dict(dtype=7), -1),
                                   (dict(temperature=0.0), -1), (dict(temperature=float("inf")), -1), (dict(temperature=2e6), -1), (dict(logits=None), -1),
                                   (dict(values=None), -1), (dict(width=1 << 20, ld=1 << 20), -4), (dict(rows=0), 0)])
def test_distill_arguments(kw, rc):
    assert _abi.lib().aig_distill_rows(C.byref(distill(**kw)), P, None, 0, None, 0, None) == rc
    assert _abi.lib().aig_distill_rows(C.byref(distill()), None, None, 0, None, 0, None) == -1       # nothing to compute
    assert _abi.lib().aig_distill_rows(C.byref(distill()), P, P, 7, None, 0, None) == -1             # rows of the gradient overlap
    assert _abi.lib().aig_distill_rows(C.byref(distill()), P, P, 8, P, 2, None) == -1


def test_sum_rows_workspace():
    lib = _abi.lib()
    assert lib.aig_sum_rows_ws_bytes(100) == 0 and lib.aig_sum_rows_ws_bytes(10 ** 7) > 0
    assert lib.aig_sum_rows(10 ** 7, P, 1.0, P, None, 0, None) == -2
    assert lib.aig_sum_rows(-1, P, 1.0, P, None, 0, None) == -1


@pytest.mark.parametrize("kw,rc", [(dict(rows=-1), -1), (dict(kinds=0), -1), (dict(classes=0), -1), (dict(classes=1025), -4),
                                   (dict(kinds=1 << 21), -4), (dict(rows=1 << 30, width=1024), -4), (dict(cand=None), -1)])
def test_class_scores_arguments(kw, rc):
    a = _abi.ScoreWindowsArg(rows=4, width=8, nodes=5, kinds=2, classes=3, cand=4096, cls=4096, row_kind=4096, by_kind=4096, kind_start=4096)
    for k, v in kw.items():
        setattr(a, k, v)
    assert _abi.lib().aig_class_scores(C.byref(a), P, P, None) == rc
    assert _abi.lib().aig_class_scores_bwd(C.byref(a), P, P, P, 1 << 40, None) == rc


def test_class_scores_workspace_is_checked():
    a = _abi.ScoreWindowsArg(rows=4000, width=8, nodes=5, kinds=2, classes=3, cand=4096, cls=4096, row_kind=4096, by_kind=4096, kind_start=4096)
    need = _abi.lib().aig_class_scores_bwd_ws_bytes(4000, 8, 2, 3)
    assert need > 0 and _abi.lib().aig_class_scores_bwd(C.byref(a), P, P, P, need - 1, None) == -2


def test_sampling_flags():
    from gan_amd.sample import build_parser, sampling_of
    base = ["--dataset-dir", "d", "--gen-ckpt", "g", "--out", "o"]
    parse = lambda *a: sampling_of(build_parser().parse_args(base + list(a)))
    assert parse() is None
    assert parse("--temperature", "0.5") == L.Sampling(0.5, 0, 1.0, 0.0)
    assert parse("--top-k", "4") == L.Sampling(1.0, 4, 1.0, 0.0)
    assert parse("--temperature", "0", "--top-p", "0.9", "--min-p", "0.1") == L.Sampling(0.0, 0, 0.9, 0.1)
    for bad in (("--temperature", "-1"), ("--temperature", "nan"), ("--top-k", "-2"), ("--top-p", "1.5"), ("--min-p", "-0.1")):
        with pytest.raises(SystemExit):
            parse(*bad)


def test_a_backward_pass_is_not_recorded(monkeypatch):
    with torch.no_grad():
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        L._check_backward("distill_loss")
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(_abi.AigAbiError, match="not recorded"):
            L._check_backward("distill_loss")


@pytest.mark.parametrize("flag,value", [("distill_top", 0), ("distill_top", 257), ("distill_temperature", 0.0), ("distill_temperature", float("nan")),
                                        ("distill_weight", -1.0), ("distill_weight", float("inf")), ("teacher_candidate_k", 0)])
def test_flags_of_a_teacher(flag, value):
    from gan_amd import train
    args = train.build_parser().parse_args(["--dataset-dir", "d", "--teacher-ckpt", "g.pt"])
    train.check_distillation(args)
    setattr(args, flag, value)
    with pytest.raises(ValueError, match=flag.replace("_", "-")):
        train.check_distillation(args)
