"""Drawn fan-ins and a generator that learns: the operators on rows of logits where the generator, the training step and the
two command lines use them."""
import ctypes as C
import math
import os

import numpy as np
import pytest
import torch

from gan_amd import _abi
from gan_amd import logits as L
from gan_amd import sample as sample_cli
from gan_amd import train as train_cli
from gan_amd.data import Data
from gan_amd.dataset import save_data_list_as_pt
from gan_amd.generator import AIGGenerator
from gan_amd.synth import synth_aig
from util_rows import distill_row, sample_row, top_row

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def generator(K, seed=0, scale=4.0, **kw):
    torch.manual_seed(seed)
    G = AIGGenerator(candidate_k=K, **kw)
    with torch.no_grad():
        for p in G.parameters():      # (logits that differ: the default initialisation is nearly flat)
            p.mul_(scale) if p.dim() > 1 else None
    return G.to(DEV).eval()


def template(n_and, seed, **kw):
    g = synth_aig(5, n_and, 3, seed=seed, window=20, orientation="dataset", **kw)
    return Data(x=g.x.to(DEV), node_depth=g.node_depth.to(DEV))


def same_graph(a, b):
    return torch.equal(a.edge_index, b.edge_index) and torch.equal(a.edge_attr.reshape(-1), b.edge_attr.reshape(-1)) and torch.equal(a.x, b.x)


@pytest.mark.parametrize("K,how", [(16, dict(temperature=1.0)), (64, dict(temperature=0.7, top_k=8, top_p=0.9)), (300, dict(min_p=0.2)),
                                   (5, dict(temperature=0.0)), (1, dict())])
@pytest.mark.parametrize("score_dtype", ["fp32", "bf16"])
def test_drawn_fan_ins(K, how, score_dtype):
    """Every slot's picks are those of its own logits; edges and bits follow the picks."""
    G, tpl = generator(K, score_dtype=score_dtype), template(120, seed=3)
    n = tpl.x.size(0)
    g = torch.Generator().manual_seed(K)
    z, u = torch.randn(128, generator=g).to(DEV), torch.rand(n, 2, generator=g).to(DEV)
    out = G(tpl, z, return_debug=True, sampling=L.Sampling(**how), u=u)
    plan, logits, sel = out._debug["plan"], out._debug["logits"].cpu().double().numpy(), out._debug["sel"].cpu().numpy()
    cnt, want, cand, order = (getattr(plan, k).cpu().numpy() for k in ("cnt", "want", "cand", "order"))
    edges, at = out.edge_index.cpu().numpy(), 0
    for r in range(n):
        if want[r] == 0:
            continue
        if cnt[r]:
            picks = sample_row(logits[r, :cnt[r]], u[r].cpu().numpy().astype(np.float64), **how)
            first = picks[0]
            second = first if want[r] < 2 or picks[1] < 0 else picks[1]
            assert list(sel[r]) == [first, second], (r, cnt[r], list(sel[r]), picks)
            sources = [cand[r, first], cand[r, second if min(want[r], cnt[r]) == 2 else first]]
        else:
            fb = int(plan.fb[r])
            sources = [fb, fb] if fb >= 0 else []
        for j in range(min(int(want[r]), len(sources))):
            assert edges[0, at] == sources[j] and edges[1, at] == order[r]
            at += 1
    assert at == edges.shape[1]
    assert same_graph(out, G(tpl, z, sampling=L.Sampling(**how), u=u))
    G.class_limit = 0                          # by node: the same logits, the same picks
    assert same_graph(out, G(tpl, z, sampling=L.Sampling(**how), u=u))
    G.class_limit = 1024
    assert G(tpl, z, sampling=L.Sampling(**how)).edge_index.shape == out.edge_index.shape       # random numbers of its own


def test_drawn_sets_are_the_single_graphs():
    G, tpl = generator(32), template(200, seed=5)
    n, S, how = tpl.x.size(0), 5, L.Sampling(temperature=0.8, top_p=0.95)
    g = torch.Generator().manual_seed(1)
    zs, us = torch.randn(S, 128, generator=g).to(DEV), torch.rand(S, n, 2, generator=g).to(DEV)
    one = G.forward_set(tpl, zs, sampling=how, u=us)
    several = [template(200, seed=50 + i) for i in range(S)]
    many = G.forward_set(several, zs, sampling=how, u=us)
    rows = L.Sampling(temperature=torch.linspace(0.2, 2.0, S * n, device=DEV), top_k=torch.full((S * n,), 6, dtype=torch.int32, device=DEV))
    each = G.forward_set(tpl, zs, sampling=rows, u=us)
    for i in range(S):
        assert same_graph(one.graph(i), G(tpl, zs[i], sampling=how, u=us[i]))
        assert same_graph(many.graph(i), G(several[i], zs[i], sampling=how, u=us[i]))
        part = slice(i * n, (i + 1) * n)
        assert same_graph(each.graph(i), G(tpl, zs[i], u=us[i], sampling=L.Sampling(rows.temperature[part].clone(), rows.top_k[part].clone())))
    sets = list(sample_cli.sample_sets(G, tpl, [(zs[:2], us[:2]), (zs[2:], us[2:])], sampling=how))
    flat = [s.graph(i) for s in sets for i in range(s.B)]
    single = list(sample_cli.sample_many(G, ((tpl, (lambda i=i: (zs[i], us[i]))) for i in range(S)), sampling=how))
    for i in range(S):
        ref = sample_cli.sample_one(G, tpl, zs[i], how, us[i])
        assert same_graph(ref, flat[i]) and same_graph(ref, single[i])


def test_drawn_fan_ins_are_refused():
    G, tpl = generator(8), template(30, seed=1)
    n, z = tpl.x.size(0), torch.zeros(128, device=DEV)
    with pytest.raises(TypeError):
        G(tpl, z, sampling=1.0)
    for u in (torch.zeros(n, 1, device=DEV), torch.zeros(n, 2), torch.zeros(n, 2, device=DEV, dtype=torch.float64)):
        with pytest.raises(_abi.AigAbiError):
            G(tpl, z, sampling=L.Sampling(), u=u)
    with pytest.raises(ValueError):
        G(tpl, z, sampling=L.Sampling(temperature=-1.0))
    a = _abi.GenWireSet()
    assert _abi.lib().aig_gen_wire_batch_sampled(C.byref(a), None, None, None) == -1
    distinct = Data(x=torch.stack([torch.randint(0, 3, (600,)).float(), torch.arange(600).float()], 1).to(DEV))
    with pytest.raises(ValueError):            # more kinds of nodes than the logits are differentiated for
        G.candidate_logits([distinct], z[None])


def test_random_numbers_of_another_shape_are_refused():
    G, tpl = generator(8), template(30, seed=1)
    n, z = tpl.x.size(0), torch.zeros(128, device=DEV)
    for shape in ((2, n), (2 * n,), (n, 2, 1)):
        with pytest.raises(_abi.AigAbiError):
            G(tpl, z, sampling=L.Sampling(), u=torch.zeros(shape, device=DEV))
    assert same_graph(G(tpl, z, sampling=L.Sampling(), u=torch.zeros(n, 2, device=DEV)),
                      G(tpl, z, sampling=L.Sampling(), u=torch.zeros(1, n, 2, device=DEV)))


def test_windows_are_kept_with_the_plans_they_are_made_of():
    G, a, b = generator(8), template(30, seed=1), template(30, seed=2)
    for templates in ([a], [a, b]):
        first, again = G.score_windows(templates), G.score_windows(templates)
        assert first[0] is again[0] and first[1] is again[1]
    assert not torch.equal(G.score_windows([a])[0].cls, G.score_windows([b])[0].cls)
    z = torch.zeros(128, device=DEV)
    before = G.candidate_logits([a], z[None]).detach()
    other = Data(x=a.x.flip(0).contiguous(), node_depth=a.node_depth)
    assert not torch.equal(G.candidate_logits([other], z[None]).detach(), before)
    assert torch.equal(G.candidate_logits([a], z[None]).detach(), before)


def reference_table(G, x_cls, z):
    """The score table in 64 bits on the CPU: ``[C, C]`` over (target class, candidate class)."""
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in G.named_parameters()}
    lin = lambda v, name: v @ p[name + ".weight"].t() + p[name + ".bias"]
    C = x_cls.size(0)
    zz = z.double().cpu().expand(C, -1)
    h = torch.relu(lin(torch.relu(lin(x_cls.double().cpu(), "node_enc.0")), "node_enc.2"))
    h = torch.relu(lin(torch.relu(lin(torch.cat([h, zz], 1), "node_proj.0")), "node_proj.2"))
    src, tgt = h.unsqueeze(0).expand(C, C, -1), h.unsqueeze(1).expand(C, C, -1)
    pair = torch.cat([src, tgt, zz.unsqueeze(0).expand(C, C, -1)], dim=2)
    return lin(torch.relu(lin(pair, "edge_scorer.0")), "edge_scorer.2")[:, :, 0], p


def test_candidate_logits_are_the_generators():
    G = generator(40)
    tpls = [template(150, seed=20 + i) for i in range(3)]
    zs = torch.randn(3, 128, generator=torch.Generator().manual_seed(2)).to(DEV)
    got = G.candidate_logits(tpls, zs).detach()
    n = tpls[0].x.size(0)
    for i, t in enumerate(tpls):
        out = G(t, zs[i], return_debug=True)
        plan, want = out._debug["plan"], out._debug["logits"]
        rows = got[i * n:(i + 1) * n]
        ok = (torch.arange(40, device=DEV) < plan.cnt[:, None])
        assert (rows[~ok] == -math.inf).all()
        ok &= plan.want[:, None] > 0
        scale = want[ok].abs().max()
        assert (rows[ok] - want[ok]).abs().max() <= 1e-5 * scale      # (both are chains of 32-bit products over 128 to 384 channels)


@pytest.mark.parametrize("k_teacher", [24, 60, 10])
def test_gradient_of_the_distillation_step(k_teacher, tmp_path):
    """The whole chain - teacher, top logits, loss, score table, parameters - against 64 bits."""
    K, t, m = 24, 2.0, 6
    teacher = generator(k_teacher, seed=9)
    torch.save(teacher.state_dict(), tmp_path / "teacher.pt")
    args = train_cli.build_parser().parse_args(["--dataset-dir", "x", "--candidate-k", str(K), "--teacher-ckpt", str(tmp_path / "teacher.pt"),
                                                "--teacher-candidate-k", str(k_teacher), "--distill-top", str(m), "--distill-temperature", str(t)])
    tr = train_cli.Trainer(args, 100, 200, DEV)
    tr.G.load_state_dict(generator(K, seed=4).state_dict())
    tpls = [template(60, seed=31), template(60, seed=32), template(45, seed=33)]
    zs = [torch.randn(128, generator=torch.Generator().manual_seed(i)).to(DEV) for i in range(3)]
    tr.opt_G.zero_grad()
    loss = tr.distill_loss(tpls, zs)
    total, grads = 0.0, {}
    for tpl, z, share in zip(tpls, zs, (1 / 3, 1 / 3, 1 / 3)):
        G = tr.G
        plan = G.plan_for(tpl, tpl.x, tpl.node_depth)
        theirs = teacher.plan_for(tpl, tpl.x, tpl.node_depth)
        S, p = reference_table(G, plan.x_cls, z)
        T, _ = reference_table(teacher, theirs.x_cls, z)
        cls, order = plan.cls.cpu().numpy(), plan.order.cpu().numpy()
        Tn, Sn = T.detach().numpy(), S.detach().numpy()
        need = [r for r in range(plan.n) if int(plan.want[r]) > 0 and int(plan.cnt[r]) > 0]
        # (templates of one size share a mean over their slots)
        group = [q for q in tpls if q.x.size(0) == tpl.x.size(0)]
        slots = sum(int(((pl.want > 0) & (pl.cnt > 0)).sum()) for pl in (G.plan_for(q, q.x, q.node_depth) for q in group))
        dS = np.zeros_like(Sn)
        for r in need:
            cs, ct = int(plan.cnt[r]), int(theirs.cnt[r])
            b = cls[order[r]]
            mine = cls[plan.cand[r, :cs].cpu().numpy()]
            x = Sn[b, mine]
            v, i, lse = top_row(Tn[b, cls[theirs.cand[r, :ct].cpu().numpy()]], min(m, k_teacher), t)
            i = np.where(i >= 0, i - (ct - cs), -1)
            l, g, _, _ = distill_row(x, v, i, lse if k_teacher == K else None, t)
            w = len(group) * share / slots
            total += w * l
            np.add.at(dS, (np.full(cs, b), mine), w * g)
        S.backward(torch.from_numpy(dS))
        for k, q in p.items():
            if q.grad is not None:
                grads[k] = grads.get(k, 0) + q.grad
    # ties: equal logits of the teacher are told apart by rounding alone (its 32-bit table against the 64-bit one), which moves
    # probability between places of one class - the table's gradient sums over them, so it stays as it is
    assert abs(float(loss) - total) <= 2e-4 * abs(total)
    for k, q in tr.G.named_parameters():
        if k.startswith("edge_attr_pred"):
            assert q.grad is None
        elif k == "edge_scorer.2.bias":        # a shift of all logits changes nothing: 0, out of terms whose sizes sum to at most 2 t,
            assert abs(float(q.grad)) <= 2 * t * 100 * 2.0 ** -24      # each off by at most 100 half steps (8 |y| + 16, |y| to 10)
        else:
            assert (q.grad.cpu().double() - grads[k]).norm() <= 2e-4 * grads[k].norm() + 1e-9, k
    before = {k: v.detach().clone() for k, v in tr.G.named_parameters()}
    tr.opt_G.step()
    assert not torch.equal(before["edge_scorer.0.weight"], tr.G.edge_scorer[0].weight)


def test_a_student_equal_to_its_teacher_has_nothing_to_learn(tmp_path):
    G = generator(32, seed=6)
    torch.save(G.state_dict(), tmp_path / "t.pt")
    args = train_cli.build_parser().parse_args(["--dataset-dir", "x", "--candidate-k", "32", "--teacher-ckpt", str(tmp_path / "t.pt")])
    tr = train_cli.Trainer(args, 100, 200, DEV)
    tr.G.load_state_dict(G.state_dict())
    loss = tr.distill_loss([template(80, seed=8)], [torch.randn(128, device=DEV)])
    # probabilities that are equal but for 32-bit roundings: the loss is of the order of their square times a logarithm, the
    # gradient of their order (2^-24 a rounding, a few dozen of them), against logits of the order of 10
    assert abs(float(loss)) <= 1e-4
    assert all(p.grad is None or p.grad.abs().max() <= 1e-3 for p in tr.G.parameters())
    bad = AIGGenerator(candidate_k=8, z_dim=40)
    torch.save(bad.state_dict(), tmp_path / "b.pt")
    args.teacher_ckpt = str(tmp_path / "b.pt")
    with pytest.raises(ValueError):
        train_cli.Trainer(args, 100, 200, DEV)


@pytest.fixture(scope="module")
def dataset(tmp_path_factory):
    root = tmp_path_factory.mktemp("distill")
    ds = root / "dataset"
    save_data_list_as_pt([synth_aig(5 + i, 30 + 8 * i, 3, seed=700 + i, window=12, orientation="dataset") for i in range(4)], str(ds), prefix="g")
    torch.save(generator(24, seed=2).state_dict(), root / "teacher.pt")
    return root, ds


@pytest.mark.parametrize("extra", [[], ["--no-sets"], ["--teacher-candidate-k", "12", "--unpad-templates"], ["--no-graph-capture"]])
def test_training_with_a_teacher(dataset, extra, capsys):
    root, ds = dataset
    out = root / ("out" + "_".join(extra).replace("-", ""))
    cwd = os.getcwd()
    os.chdir(root)
    try:
        train_cli.main(["--dataset-dir", str(ds), "--out-dir", str(out), "--epochs", "1", "--batch-size", "2", "--candidate-k", "24",
                        "--seed", "5", "--no-progress", "--teacher-ckpt", str(root / "teacher.pt"), "--distill-top", "8"] + extra)
    finally:
        os.chdir(cwd)
    said = capsys.readouterr().out
    assert "distillation loss" in said and "[ERROR]" not in said
    torch.manual_seed(5)
    init = AIGGenerator(candidate_k=24).state_dict()
    moved = torch.load(out / "generator_epoch0.pt", weights_only=True)
    assert all(torch.isfinite(v).all() for v in moved.values())
    for k in init:
        same = torch.equal(init[k], moved[k].cpu())
        assert same if k.startswith("edge_attr_pred") else not same or k == "edge_scorer.2.bias", k
    if not extra:        # the critic's side of the first step is what it is without a teacher
        plain = root / "plain"
        os.chdir(root)
        try:
            train_cli.main(["--dataset-dir", str(ds), "--out-dir", str(plain), "--epochs", "1", "--batch-size", "2", "--candidate-k", "24",
                            "--seed", "5", "--no-progress"])
        finally:
            os.chdir(cwd)
        rows = [open(d / "metrics.csv").read().splitlines()[1] for d in (out, plain)]
        assert rows[0] == rows[1]


def test_sampling_command_line_with_drawn_fan_ins(dataset):
    root, ds = dataset
    base = ["--dataset-dir", str(ds), "--gen-ckpt", str(root / "teacher.pt"), "--candidate-k", "24", "--seed", "9", "--temperature", "0.9",
            "--top-p", "0.95"]
    for name, extra in (("a", ["--num-samples", "5"]), ("b", ["--num-samples", "5", "--batch", "1"]), ("c", ["--num-samples", "5", "--batch", "2"])):
        sample_cli.main(base + ["--out", str(root / name / "s.pt")] + extra)
    picks = {name: [torch.load(root / name / f"s_{i:06d}.pt", weights_only=True) for i in range(5)] for name in "abc"}
    for i in range(5):
        for name in "bc":
            assert all(torch.equal(picks["a"][i][k], picks[name][i][k]) for k in picks["a"][i])
    assert any(not torch.equal(picks["a"][0]["edge_index"], picks["a"][i]["edge_index"]) for i in range(1, 5))
    sample_cli.main(base + ["--out", str(root / "one.pt")])
    one = torch.load(root / "one.pt", weights_only=True)
    assert all(torch.equal(one[k], picks["a"][0][k]) for k in one)
    with pytest.raises(SystemExit):
        sample_cli.main(base + ["--out", str(root / "x.pt"), "--min-p", "2"])
