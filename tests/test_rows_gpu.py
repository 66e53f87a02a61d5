"""Rows of logits: calls that their operators once answered wrongly, against definitions in 64 bits."""
import copy

import pytest
import torch

from gan_amd import _abi
from gan_amd import logits as L
from gan_amd import train as train_cli
from gan_amd.data import Batch
from gan_amd.dataset import pad_data
from gan_amd.synth import synth_aig
from test_distill_gpu import generator, template
from test_logits_gpu import BF16, F16, F32, check_distill, check_sample, make_logits, make_windows, rng
from util_rows import sample_row

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.mark.parametrize("rows,width", [(300, 9), (300, 20), (300, 64), (200, 256), (100, 512), (100, 1024), (12, 1500), (530, 2048)])
def test_places_of_little_weight_are_drawn_when_they_are_what_is_left(rows, width):
    """Few places, most of them far below the largest: once the largest is drawn, what is left is below the last bit of the
    sum that held it - and is drawn all the same."""
    g = rng(width)
    counts = torch.randint(2, min(width, 8) + 1, (rows,), generator=g, dtype=torch.int32)
    u = torch.rand(rows, 4, generator=g)
    for i, t in enumerate((0.05, 0.1, 0.2, 0.3)):
        x = make_logits(rows, width, (F32, BF16, F16)[i % 3], seed=width + i)
        x[0, :2] = torch.tensor([0.0, -18.0 * t])          # one place beside the largest, in the same lane
        counts[0] = 2
        x[1] = -50.0                                       # ... at the lane's end, and in the one beside it
        x[1, :8] = torch.tensor([0.0, -17.0, -17.5, -18.0, -19.0, -20.0, -21.0, -22.0]) * t
        counts[1] = min(8, width)
        x[2, :2] = torch.tensor([0.0, -26.0]) * t          # below a multiple of 2^-36: nothing is left
        counts[2] = 2
        x[3, :3] = torch.tensor([0.0, -24.5, -24.0]) * t
        counts[3] = 3
        for how in (dict(), dict(top_k=2), dict(top_k=3)):
            check_sample(x, u, counts=counts, temperature=t, **how)
    # all of a row's places that stay in one lane, among many that do not
    x = make_logits(rows, width, F32, seed=3) - 8.0
    x[:, 0], x[:, 1], x[:, 2] = 9.0, -8.0, -8.5
    x[:, 3:] -= 20.0
    check_sample(x, u, top_k=3)
    check_sample(x, u[:, :2].contiguous(), top_k=2)
    check_sample(x, u)


@pytest.mark.parametrize("rows,width", [(400, 9), (400, 64), (200, 256), (100, 512), (100, 1024), (12, 1500), (530, 2048)])
def test_min_p_is_compared_with_weights_in_whole_units(rows, width):
    """A min-p of a few units of 2^-36: the half that a weight is rounded by decides who reaches it."""
    g, unit = rng(width + 1), 2.0 ** -36
    n = min(width, 8)
    counts = torch.full((rows,), n, dtype=torch.int32)
    u = torch.rand(rows, 4, generator=g)
    for i, share in enumerate((1e-9, 68.5 * unit, 5.4 * unit, 2.5 * unit, 1.5 * unit, unit, 1e-12)):
        x = make_logits(rows, width, F32, seed=width + i)
        # weights from a little under the share to a little over it, beside the largest
        x[:, :n] = torch.log(torch.tensor(share * 0.98)) + 0.04 * torch.rand(rows, n, generator=g)
        x[:, 0] = 0.0
        x[: rows // 2, 1:n] = torch.log(torch.tensor(share)) + 0.6 * (torch.rand(rows // 2, n - 1, generator=g) - 0.5)
        check_sample(x, u, counts=counts, min_p=share)
        check_sample(x, u, counts=counts, min_p=share, top_k=5)


@pytest.mark.parametrize("K,n_and", [(8, 150), (40, 150), (300, 150), (700, 1100), (1024, 1600)])
def test_fan_ins_drawn_at_a_low_temperature(K, n_and):
    """A slot's second fan-in is its second draw, however little of the weight that has."""
    G, tpl = generator(K, seed=3), template(n_and, seed=4)
    n, g = tpl.x.size(0), rng(K)
    z, u = torch.randn(128, generator=g).to(DEV), torch.rand(n, 2, generator=g).to(DEV)
    logits = G(tpl, z, return_debug=True, sampling=L.Sampling(), u=u)._debug["logits"].cpu().double()
    plan = G.plan_for(tpl, tpl.x, tpl.node_depth)
    cnt, want = plan.cnt.cpu(), plan.want.cpu()
    t = torch.ones(n)
    for r in range(n):                       # what is below the largest logit of a slot has e^-20 of its weight and less
        v = logits[r, :cnt[r]].unique()
        t[r] = (v[-1] - v[-2]) / 20.0 if want[r] > 0 and len(v) > 1 else 1.0
    sel = G(tpl, z, return_debug=True, sampling=L.Sampling(temperature=t.to(DEV)), u=u)._debug["sel"].cpu()
    seconds = 0
    for r in range(n):
        if want[r] == 0 or cnt[r] == 0:
            continue
        first, second = sample_row(logits[r, :cnt[r]].numpy(), u[r].double().cpu().numpy(), temperature=float(t[r]))
        second = first if want[r] < 2 or second < 0 else second
        seconds += first != second
        assert sel[r].tolist() == [first, second], (r, int(cnt[r]), float(t[r]))
    assert seconds > 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(9, 64), (9, 300), (530, 2000), (9, 2000), (5, 5000)])
def test_gradient_of_logits_that_hooks_hand_back_as_copies(rows, width, dtype):
    """Saved on the host, cloned, or laid out by columns: the gradient is that without hooks."""
    whole = make_logits(rows, width + 24, dtype, seed=width).to(DEV)
    whole[:, width:] = float("nan")                # (what lies beside the rows is none of theirs)
    teacher = make_logits(rows, width, F32, seed=width + 1).to(DEV)
    top = L.top_rows(teacher, 8, temperature=2.0)
    counts = torch.full((rows,), width - 1, dtype=torch.int32, device=DEV)
    weight, up = torch.rand(rows, generator=rng(1)).to(DEV), torch.randn(rows, generator=rng(2)).to(DEV)
    hooks = (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone()),
             torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t))

    def gradient(view):
        leaf = whole.detach().clone().requires_grad_(True)
        loss = L.distill_loss(view(leaf), top, counts=counts, weight=weight, temperature=2.0, reduction="none")
        return leaf, loss

    for view in (lambda v: v[:, :width], lambda v: v[:, :width].contiguous(), lambda v: v[1:2, :width].expand(rows, width)):
        leaf, loss = gradient(view)
        loss.backward(up)
        for hook in hooks:
            with hook:
                other, again = gradient(view)
            assert torch.equal(again, loss)
            again.backward(up)
            assert torch.equal(other.grad, leaf.grad)      # (a place's slope depends on its row's sums, which the loss left, alone)


def test_gradient_of_a_table_whose_windows_are_saved_elsewhere():
    cand, counts, cls, kind = make_windows(300, 40, 100, 5, 9, seed=2)
    w = L.ScoreWindows.of(*(v.to(DEV) for v in (cand, counts, cls, kind)), 5)
    table, g = torch.randn(5, 9, generator=rng(1)).to(DEV).requires_grad_(True), torch.randn(300, 40, generator=rng(2)).to(DEV)
    L.class_scores(table, w).backward(g)
    want, table.grad = table.grad, None
    for hook in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone())):
        with hook:
            out = L.class_scores(table, w)
        out.backward(g)
        assert torch.equal(table.grad, want)
        table.grad = None


@pytest.mark.parametrize("extra", [[], ["--no-graph-capture"]])
def test_a_step_that_raises_leaves_the_generator_alone(extra, tmp_path, monkeypatch):
    """A skipped step is skipped for the generator too, wherever it raised; the next one moves it."""
    graphs = [synth_aig(6, 40, 3, seed=60 + i, window=16, orientation="dataset") for i in range(2)]
    mn, me = max(g.x.size(0) for g in graphs), max(g.edge_index.size(1) for g in graphs)
    batch = Batch.from_data_list([pad_data(g, mn, me) for g in graphs]).to(DEV)
    torch.save(generator(12, seed=9).state_dict(), tmp_path / "teacher.pt")
    args = train_cli.build_parser().parse_args(["--dataset-dir", "x", "--candidate-k", "12", "--teacher-ckpt", str(tmp_path / "teacher.pt"),
                                                "--distill-top", "4", "--n-critic", "2", "--save-every", "2"] + extra)
    torch.manual_seed(3)
    tr = train_cli.Trainer(args, mn, me, DEV)
    weights = lambda: [p.detach().clone() for p in tr.G.parameters()]
    start = weights()

    def boom(*a, **k):
        raise RuntimeError("injected failure")
    with monkeypatch.context() as patch:
        patch.setattr(train_cli, "validate_strict_aig", boom)          # (behind the distillation and the generator's pass)
        with pytest.raises(RuntimeError, match="injected"):
            tr.step(batch)
    assert all(torch.equal(a, b) for a, b in zip(start, weights())) and not tr.opt_G.state
    with monkeypatch.context() as patch:
        patch.setattr(tr, "distill_loss", boom)
        with pytest.raises(RuntimeError, match="injected"):
            tr.step(batch)
    assert all(torch.equal(a, b) for a, b in zip(start, weights())) and not tr.opt_G.state
    tr.step(batch)
    assert any(not torch.equal(a, b) for a, b in zip(start, weights()))
    assert all(int(v["step"]) == 1 for v in tr.opt_G.state.values())


@pytest.mark.parametrize("count", [1, 3])
def test_windows_made_on_one_stream_and_read_on_another(count):
    """The second caller's stream waits for what the first caller's has been given to make."""
    G, tpls = generator(24), [template(400, seed=70 + i) for i in range(count)]
    z = torch.randn(count, 128, generator=rng(4)).to(DEV)
    fresh = generator(24)
    want = fresh.candidate_logits([t.clone() for t in tpls], z).detach()
    G._stacked_plans(tpls, DEV)                     # (the plans themselves are there)
    busy = torch.zeros(1 << 28, device=DEV)
    torch.cuda.synchronize()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(first):
        for _ in range(60):                         # (some 30 ms)
            busy.add_(1.0)
        mine = G.score_windows(tpls)
    assert not first.query()
    with torch.cuda.stream(second), torch.no_grad():
        theirs = G.score_windows(tpls)
        got = G.candidate_logits(tpls, z)
        assert theirs[0] is mine[0]
    second.synchronize()
    assert torch.equal(got, want)
    again = G.candidate_logits(tpls, z).detach()
    assert torch.equal(again, want)


@pytest.mark.parametrize("count", [1, 2])
def test_candidate_logits_in_a_recording(count):
    """Windows are made in front of a recording; what is recorded then follows z."""
    G, tpls = generator(24), [template(60, seed=80 + i) for i in range(count)]
    z = torch.randn(count, 128, generator=rng(5)).to(DEV)
    graph = torch.cuda.CUDAGraph()
    G._stacked_plans(tpls, DEV)
    torch.cuda.synchronize()
    with torch.no_grad():
        with torch.cuda.graph(graph, capture_error_mode="thread_local"):
            with pytest.raises(_abi.AigAbiError, match="in front of a recording"):
                G.score_windows(tpls)
            kept = z * 2.0
        for _ in range(2):
            G.candidate_logits(tpls, z)
            torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="thread_local"):
            got = G.candidate_logits(tpls, z)
        for k in range(3):
            z.copy_(torch.randn(count, 128, generator=rng(6 + k)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, G.candidate_logits(tpls, z)), k


def test_windows_of_one_template_hold_no_second_copy_of_its_candidates():
    G, a, b = generator(24), template(60, seed=1), template(60, seed=2)
    plan = G.plan_for(a, a.x, a.node_depth)
    windows = G.score_windows([a])[0]
    assert windows.cand.data_ptr() == plan.cand.data_ptr() and windows.cand.shape == (plan.n, 24)
    both = G.score_windows([a, b])[0].cand
    other = G.score_windows([b])[0].cand
    for r in range(plan.n):                     # (past a row's count a window holds whatever it did)
        k = int(plan.cnt[r])
        assert torch.equal(both[r, :k], windows.cand[r, :k])
    cnt = G.plan_for(b, b.x, b.node_depth).cnt
    for r in range(plan.n):
        assert torch.equal(both[plan.n + r, :cnt[r]], other[r, :cnt[r]] + plan.n)


@pytest.mark.parametrize("rows,width", [(6, 7), (6, 16), (6, 60), (6, 200), (6, 500), (6, 1000), (6, 1500), (530, 2000)])
def test_listed_places_without_probability(rows, width):
    """A teacher's masked places that are listed all the same: they are not of the rest, and a student's masked place has no
    gradient."""
    low = torch.finfo(F32).min
    x = make_logits(rows, width, F32, seed=width)
    i = torch.arange(6, dtype=torch.int32).expand(rows, 6).contiguous()
    v = x[:, :6] + 0.5 * torch.randn(rows, 6, generator=rng(2))
    x[:, 3:5], v[:, 3:5] = low, low
    v[:, 5] = -200.0                              # no probability, but a student's that is not masked
    s = torch.logsumexp(v.double() / 1.5, 1).float() + 0.5
    for lse in (s, None):
        _, grad = check_distill(x[:8], v[:8], i[:8], None if lse is None else lse[:8], 1.5)
        assert not grad[:, 3:5].any()
    _, grad = L.distill_loss_and_grad(x.to(DEV), L.TopRows(v.to(DEV), i.to(DEV), s.to(DEV)), temperature=1.5)
    assert not grad[:, 3:5].any() and grad[:, 5].all()


@pytest.mark.parametrize("width", [5, 48, 200, 500, 1000, 1500])
def test_probabilities_of_many_entries_of_one_place_add_up(width):
    """256 entries whose probabilities lie between the steps of 2^-23: their sum is not off by 256 half steps."""
    x = make_logits(4, width, F32, seed=width)
    i = torch.full((4, 256), 3, dtype=torch.int32)
    q = (torch.arange(92000, 92004).double()[:, None] + torch.tensor([0.45, 0.48, 0.49, 0.47]).double()[:, None]) * 2.0 ** -23
    v = torch.log(q).expand(4, 256).float().clone()
    v[:, 0] = 0.0
    v[:, 1] = 0.0
    i[:, 1] = 1
    s = torch.zeros(4)
    check_distill(x, v, i, s, 1.0)
    check_distill(x, v, i, None, 1.0)


def test_a_template_with_windows_can_be_copied():
    G, tpl, z = generator(24), template(60, seed=1), torch.randn(1, 128, generator=rng(2)).to(DEV)
    want = G.candidate_logits([tpl], z).detach()
    other = copy.deepcopy(tpl)
    assert torch.equal(G.candidate_logits([other], z).detach(), want)


@pytest.mark.parametrize("count", [1, 2])
def test_templates_that_were_sampled_in_inference_mode_can_be_trained_on(count):
    tpls, z = [template(50, seed=1 + i) for i in range(count)], torch.randn(count, 128, generator=rng(3)).to(DEV)
    grads = []
    for first in (True, False):
        G = generator(16)
        here = tpls if first else [t.clone() for t in tpls]
        if first:
            with torch.inference_mode():
                G(here[0], z[0]), G.forward_set(here, z), G.candidate_logits(here, z)
        G.candidate_logits(here, z).nan_to_num(neginf=0.0).square().sum().backward()
        grads.append([p.grad for p in G.parameters()])
    assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(*grads))
    assert any(g is not None and g.any() for g in grads[0])


@pytest.mark.parametrize("width", [40, 5000])
def test_a_teacher_that_was_asked_in_inference_mode(width):
    x = make_logits(30, width, F32, seed=1).to(DEV).requires_grad_(True)
    cand, counts, cls, kind = (v.to(DEV) for v in make_windows(30, width, 100, 5, 9, seed=2))
    table = torch.randn(5, 9, generator=rng(4)).to(DEV).requires_grad_(True)

    def asked():
        teacher = make_logits(30, width, F32, seed=2).to(DEV)
        c, weight = counts.clone(), torch.rand(30, generator=rng(3)).to(DEV)
        return L.top_rows(teacher, 8, counts=c, temperature=2.0), c, weight, L.ScoreWindows.of(cand, c, cls, kind, 5)

    grads = []
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            top, c, weight, windows = asked()
        L.distill_loss(x, top, counts=c, weight=weight, temperature=2.0).backward()
        L.distill_loss(L.class_scores(table, windows), top, counts=c, temperature=2.0).backward()
        grads.append((x.grad, table.grad))
        x.grad = table.grad = None
    assert all(torch.equal(a, b) and a.any() for a, b in zip(*grads))


def test_windows_that_are_let_go_while_another_stream_reads_them():
    """Their memory is not given to others before that stream is through."""
    G, z = generator(24), torch.randn(2, 128, generator=rng(4)).to(DEV)
    tpls = [template(3000, seed=90 + i) for i in range(2)]
    want = generator(24).candidate_logits([t.clone() for t in tpls], z).detach()
    windows, weight, _ = G.score_windows(tpls)
    sizes = {v.data_ptr(): v.numel() for v in (*windows, weight)}
    busy = torch.zeros(1 << 28, device=DEV)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other), torch.no_grad():
        for _ in range(60):                         # (some 30 ms)
            busy.add_(1.0)
        got = G.candidate_logits(tpls, z)
    del windows, weight, tpls
    G.__dict__["_plan_stacks"].clear()
    mine = [torch.full((n,), -1, dtype=torch.int32, device=DEV) for n in sizes.values() for _ in range(3)]
    assert not other.query()
    assert not {v.data_ptr() for v in mine} & set(sizes)
    other.synchronize()
    assert torch.equal(got, want)
