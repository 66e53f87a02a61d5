"""Two data-parallel ranks of ``Trainer.step`` with a teacher (not collected by pytest: started by tests/conftest.py before
the test session touches the GPU, checked by tests/test_parallel_teacher_gpu.py).

    python -m torch.distributed.run --nnodes=1 --nproc-per-node=2 ... tests/dp_teacher.py OUT.json

The ranks share one GPU (``AIG_DIST_BACKEND=gloo``).  OUT.json:

  grad_mean_err   the exchanged gradient of the generator against the mean of what each rank's minibatch gives alone
  steps           by where rank 1's step raises (nothing: nowhere; both: in both ranks): are generator and critic of
                  the two ranks equal afterwards, how far the generator moved, what each rank's step raised
"""
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))

import torch
import torch.distributed as dist

from dp_rehearsal import WATCH, flat, start_watchdog
from gan_amd import parallel
from gan_amd.data import Batch
from gan_amd.dataset import pad_data
from gan_amd.generator import AIGGenerator
from gan_amd.synth import synth_aig
from gan_amd.train import Trainer, build_parser


def boom(*a, **k):
    raise RuntimeError("injected failure")


def main():
    out_path = sys.argv[1]
    rank, local_rank, world = parallel.init_distributed()
    start_watchdog(rank, 80.0)
    assert world == 2, "written for two ranks"
    dev = torch.device("cuda", local_rank % max(torch.cuda.device_count(), 1))
    torch.cuda.set_device(dev)
    graphs = [synth_aig(6 + i, 40 + 10 * i, 4, seed=50 + i, window=16, orientation="dataset") for i in range(2)]
    mn, me = max(g.x.size(0) for g in graphs), max(g.edge_index.size(1) for g in graphs)
    batches = [Batch.from_data_list([pad_data(g, mn, me)]).to(dev) for g in graphs]
    for i, b in enumerate(batches):
        b.sample_ids = [i]
    ckpt = f"{out_path}.teacher{rank}.pt"
    torch.manual_seed(9)
    teacher = AIGGenerator(candidate_k=16)
    with torch.no_grad():
        for p in teacher.parameters():
            p.mul_(4.0) if p.dim() > 1 else None
    torch.save(teacher.state_dict(), ckpt)
    flags = ["--dataset-dir", "unused", "--candidate-k", "16", "--n-critic", "2", "--save-every", "1000", "--teacher-ckpt", ckpt,
             "--distill-top", "4"]
    torch.manual_seed(1234 + rank)
    made = {True: Trainer(build_parser().parse_args(flags), mn, me, dev, rank, world)}
    made[False] = Trainer(build_parser().parse_args(flags + ["--no-graph-capture"]), mn, me, dev, rank, world)
    g = torch.Generator().manual_seed(5)
    zs = [torch.randn(128, generator=g).to(dev) for _ in range(2)]
    for tr in made.values():
        tr.global_step = 1

    # the exchanged gradient of the first step, and what each minibatch gives by itself
    tr, alone = made[True], []
    for who in range(2):
        tr.opt_G.zero_grad()
        tr.distill_loss(tr.templates_of(batches[who]), [zs[who]])
        alone.append(torch.cat([(torch.zeros_like(p) if p.grad is None else p.grad).reshape(-1) for p in tr.G.parameters()]))
    mean = (alone[0] + alone[1]) / 2
    seen, inner = {}, tr.g_reducer.reduce

    def reduce(ok=True):
        out = inner(ok)
        seen.setdefault("g", torch.cat([p.grad.reshape(-1) for p in tr.G.parameters()]))
        return out
    tr.g_reducer.reduce = reduce

    calls = {"n": 0, "from": None}

    def draw_z():
        calls["n"] += 1
        if calls["from"] is not None and calls["n"] >= calls["from"]:
            boom()
        return zs[rank].clone()

    steps = {}

    def step(what, tr, sabotage=None):
        WATCH["trainer"], WATCH["phase"] = tr, what
        before, raised = flat(tr.G.parameters()), None
        calls.update(n=0, **{"from": None})
        tr.draw_z = draw_z
        undo = sabotage(tr) if sabotage is not None and (rank == 1 or what == "both") else None
        try:
            tr.step(batches[rank])
        except RuntimeError as e:
            raised = str(e)
        if undo is not None:
            undo()
        weights = flat(tr.G.parameters())
        mine = torch.cat([weights, flat(tr.D.parameters())])
        both = [torch.empty_like(mine) for _ in range(world)]
        dist.all_gather(both, mine)
        steps[what] = {"equal": bool(torch.equal(both[0], both[1])), "moved": float((weights - before).abs().max()), "raised": raised,
                       "finite": bool(torch.isfinite(weights).all())}
        print(f"rank {rank}: {what} {steps[what]}", flush=True)

    def draws_from(n):
        def sabotage(tr):
            calls["from"] = n
        return sabotage

    def replaced(name):
        def sabotage(tr):
            kept = getattr(tr, name)
            setattr(tr, name, boom)
            return lambda: setattr(tr, name, kept)
        return sabotage

    def generator_pass(tr):          # the pass over the raw graphs: the second one of a step
        kept, count = tr.G.forward_set, {"n": 0}

        def forward_set(*a, **k):
            count["n"] += 1
            if count["n"] >= 2:
                boom()
            return kept(*a, **k)
        tr.G.forward_set = forward_set

        def undo():
            del tr.G.forward_set
        return undo

    step("nothing", made[True])
    err = float((seen["g"] - mean).abs().max() / mean.abs().max())
    step("critic", made[True], draws_from(1))            # in front of the first gradient of the critic
    step("early draws", made[True], draws_from(2))       # ... the raw graphs' draws, where they are made early
    step("raw graphs", made[True], generator_pass)
    step("distillation", made[True], replaced("distill_loss"))
    step("draws", made[False], draws_from(2))            # between the two exchanges
    step("both", made[True], replaced("distill_loss"))   # (no rank has a gradient: zeros, and the optimiser's momentum)
    mine = {"rank": rank, "grad_mean_err": err, "steps": steps}
    gathered = [None] * world
    dist.all_gather_object(gathered, mine)
    if rank == 0:
        with open(out_path + ".tmp", "w") as f:
            json.dump(gathered, f)
        os.replace(out_path + ".tmp", out_path)
    dist.barrier()
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
