"""Sampling, top logits, distillation and class scores on rows of logits, against their definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

from gan_amd import _abi
from gan_amd import logits as L
from util_rows import distill_row, sample_row, top_row

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rng(seed):
    return torch.Generator().manual_seed(seed)


def make_logits(rows, width, dtype, seed, ties=False):
    g = rng(seed)
    if ties:
        return torch.randint(-3, 4, (rows, width), generator=g).to(dtype)
    return (2.0 * torch.randn(rows, width, generator=g)).to(dtype)


def make_counts(rows, width, seed):
    c = torch.randint(0, width + 1, (rows,), generator=rng(seed + 77), dtype=torch.int32)
    c[0] = width
    if rows > 1:
        c[1] = 0
    if rows > 2:
        c[2] = min(1, width)
    return c


def check_sample(x, u, counts=None, want=None, **how):
    dev = {k: (v.to(DEV) if torch.is_tensor(v) else v) for k, v in how.items()}
    got = L.sample_rows(x.to(DEV) if not x.is_cuda else x, u.to(DEV), counts=None if counts is None else counts.to(DEV),
                        want=None if want is None else want.to(DEV), **dev).cpu().numpy()
    xs, us = x.detach().cpu().float().numpy().astype(np.float64), u.numpy().astype(np.float64)
    for r in range(x.size(0)):
        n = x.size(1) if counts is None else min(max(int(counts[r]), 0), x.size(1))
        one = {k: (v[r].item() if torch.is_tensor(v) else v) for k, v in how.items()}
        ref = sample_row(xs[r, :n], us[r], **one)
        if want is not None:
            ref = [p if d < int(want[r]) else -1 for d, p in enumerate(ref)]
        assert list(got[r]) == ref, (r, n, one, us[r], list(got[r]), ref)
    return got


WIDTHS = [1, 2, 3, 15, 16, 17, 63, 64, 65, 100, 255, 256, 257, 511, 512, 513, 777, 1023, 1024, 1025, 1500, 8192, 8193, 20001]
SETTINGS = [dict(), dict(temperature=0.7, top_k=5), dict(temperature=1.3, top_p=0.8), dict(min_p=0.1),
            dict(temperature=0.5, top_k=20, top_p=0.9, min_p=0.02), dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0),
            dict(top_p=1e-6, temperature=3.0), dict(min_p=1.0), dict(top_k=1000000, top_p=0.999)]


@pytest.mark.parametrize("width", WIDTHS)
def test_sample_every_width(width):
    rows = 37 if width <= 1024 else 5
    for i, how in enumerate(SETTINGS):
        dtype = (F32, BF16, F16)[(i + width) % 3]
        x = make_logits(rows, width, dtype, seed=width + i, ties=i % 2 == 1)
        u = torch.rand(rows, 1 + (i + width) % 4, generator=rng(1000 + i))
        check_sample(x, u, counts=make_counts(rows, width, i) if i % 3 else None, **how)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", [7, 64, 200, 700, 3000])
def test_sample_special_values(dtype, width):
    inf, low = math.inf, torch.finfo(dtype).min
    x = make_logits(16, width, dtype, seed=3)
    x[0] = -inf                                # nothing in the row
    x[1] = low                                 # masked by the type's lowest value throughout: all alike
    x[2, 1:] = low
    x[3, ::2] = -inf
    x[4, ::3] = float("nan")                   # NaN is never drawn
    x[5] = float("nan")
    x[6, 2], x[6, width - 1] = inf, inf        # two infinities share the mass
    x[7] = 1.5
    x[8] = 0.0
    x[8, ::2] = -0.0                           # the two zeros are one value
    x[9, width // 2:] = low
    x[10] = torch.arange(width) % 3
    x[11] = -x[11].abs() * 30 - 5
    counts = torch.full((16,), width, dtype=torch.int32)
    counts[12] = 0
    counts[13], counts[14], counts[15] = width - 1, -5, width + 99      # outside: the nearer bound
    x[13, width - 1] = inf                     # past the count: not there
    for how in (dict(), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.3), dict(temperature=0.0),
                dict(temperature=0.01, top_k=3, top_p=0.7), dict(temperature=1e30), dict(temperature=1e-30)):
        for seed in (1, 2):
            check_sample(x, torch.rand(16, 3, generator=rng(seed)), counts=counts, **how)


def test_sample_edges_of_the_random_numbers():
    x = make_logits(12, 100, F32, seed=5)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan"), math.inf, -math.inf, 2.0 ** -30, 0.5, 1e-45, 0.999999])
    u = torch.stack([u, u.flip(0)], dim=1).contiguous()
    check_sample(x, u)
    check_sample(x, u, top_p=0.9)
    check_sample(make_logits(12, 2000, F32, seed=6), u, top_k=700)


def test_sample_each_row_its_settings_and_want():
    rows = 96
    g = rng(8)
    for width in (40, 300, 900, 5000):
        x = make_logits(rows if width < 1000 else 8, width, F32, seed=width, ties=True)
        n = x.size(0)
        how = dict(temperature=torch.rand(n, generator=g) * 2, top_k=torch.randint(-1, 30, (n,), generator=g, dtype=torch.int32),
                   top_p=torch.rand(n, generator=g) * 1.3, min_p=torch.rand(n, generator=g) * 0.4 - 0.1)
        how["temperature"][::5] = 0.0
        want = torch.randint(-1, 6, (n,), generator=g, dtype=torch.int32)
        check_sample(x, torch.rand(n, 4, generator=g), counts=make_counts(n, width, 1), want=want, **how)


@pytest.mark.parametrize("width,dtype,off", [(9, F32, 0), (64, BF16, 0), (300, F32, 1), (1000, F16, 0), (1025, F16, 3), (5000, F32, 0), (9001, BF16, 1)])
def test_sample_follows_the_probabilities(width, dtype, off):
    """Evenly spread random numbers hit every place as often as its probability says, to within one - and never a place
    that a filter took out."""
    N, t = 4096, 0.8
    row = make_logits(1, width + off, dtype, seed=width, ties=width == 1025)
    x = row.to(DEV)[:, off:].expand(N, width)
    v = row[0, off:].double().numpy()
    w = np.exp((v - v.max()) / np.float64(np.float32(t)))
    u = ((torch.arange(N) + 0.5) / N).reshape(N, 1)
    order = np.lexsort((np.arange(width), -v))
    for how in (dict(), dict(min_p=0.1), dict(top_k=5), dict(top_p=0.7), dict(top_p=0.7, min_p=0.2), dict(top_k=40, top_p=0.9)):
        got = L.sample_rows(x, u.to(DEV), temperature=t, **how)[:, 0].cpu().numpy()
        keep = order[:how.get("top_k", width)]
        front = np.concatenate([[0.0], np.cumsum(w[keep])[:-1]])
        keep = keep[(front < np.float64(np.float32(how["top_p"])) * w[keep].sum()) | (front == 0)] if "top_p" in how else keep
        keep = keep[w[keep] >= how.get("min_p", 0.0)]
        p = np.zeros(width)
        p[keep] = w[keep] / w[keep].sum()
        hits = np.bincount(got, minlength=width)
        assert np.all(np.abs(hits - N * p) <= 1.0 + 1e-6), how
        assert not hits[p == 0].any(), how


@pytest.mark.parametrize("width", [4, 64, 256, 512, 1024, 2048, 16384])
def test_sample_decisions_on_a_border(width):
    """Equal logits: random numbers that fall on the borders between places exactly, and a share of the mass that does."""
    x = torch.full((64, width), 0.25)
    u = (torch.arange(64) / 64.0).reshape(64, 1)
    got = check_sample(x, u)
    assert np.array_equal(got[:, 0], np.arange(64) * width // 64)
    for p in (0.25, 0.5, 0.75):
        got = check_sample(x, u, top_p=p)
        assert got.max() < p * width
    check_sample(x, u, top_k=width // 2, top_p=0.5, min_p=1.0)


@pytest.mark.parametrize("width", [20, 64, 65, 200, 256, 500, 512, 777, 1024])
def test_sample_borders_among_places_that_do_not_part(width):
    """Equal logits, logits a last bit apart, masks of the lowest value, places of no weight, one place with all of it."""
    x = make_logits(12, width, F32, seed=width)
    x[0] = 2.5
    x[1] = torch.where(torch.rand(width, generator=rng(1)) < 0.5, 2.0, 1.0)
    x[2] = 3.0 + torch.arange(width) * 2.0 ** -22
    x[3, 5:] = torch.finfo(F32).min
    x[4, 3:] = -math.inf
    x[5, 0] = 60.0
    x[6] = torch.randint(0, 4, (width,), generator=rng(2)).float()
    x[7] = -20.0
    x[7, -1] = 0.0
    x[8] = torch.linspace(0.0, -30.0, width)
    x[9] = torch.where(torch.rand(width, generator=rng(3)) < 0.7, -math.inf, 1.0)
    x[10] = 1e-7 * x[10]
    x[11, : width // 2] = x[11].max()
    u = torch.rand(12, 3, generator=rng(4))
    for k in (0, 1, 7, 16, 32, 33, 64, 65, 130):
        for p in (1.0, 0.0, 0.3, 0.9, 0.999, 1.0 - 2.0 ** -20):
            if k or p < 1:
                check_sample(x, u, top_k=k, top_p=p, temperature=0.9)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width,ld", [(1025, 1025), (1600, 1608), (2047, 2050), (2048, 2048)])
def test_many_rows_are_answered_like_few(width, ld, dtype):
    """Rows of 1025 to 2048 places: what hundreds of them get is what a part of them gets, and the first few are the oracle's."""
    rows, m, t = 530, 20, 1.5
    x = torch.empty(rows, ld, dtype=dtype)
    x[:, :width] = make_logits(rows, width, dtype, seed=width)
    x[:, width:] = float("nan")
    x = x[:, :width]
    x[0, ::2] = -math.inf
    x[1] = 1.0
    x[2] = -math.inf
    x[3, 7:] = torch.finfo(dtype).min
    x[4, ::3] = float("nan")
    x[5] = make_logits(1, width, dtype, seed=3, ties=True)[0]
    x[6, 5:] = math.inf
    counts = make_counts(rows, width, 5)
    counts[:8] = width
    u = torch.rand(rows, 2, generator=rng(6))
    dx, dc, du = x.to(DEV), counts.to(DEV), u.to(DEV)
    full = torch.empty(rows, ld, dtype=dtype, device=DEV)
    full[:, :width] = dx
    full[:, width:] = float("nan")
    dx = full[:, :width]
    parts = (slice(0, 200), slice(200, 400), slice(400, rows))
    for how in (dict(), dict(top_p=0.9), dict(top_k=50), dict(top_k=30, top_p=0.8, min_p=0.01), dict(top_k=700, temperature=0.8), dict(temperature=0.0)):
        many = L.sample_rows(dx, du, counts=dc, **how)
        few = torch.cat([L.sample_rows(dx[s], du[s].contiguous(), counts=dc[s].contiguous(), **how) for s in parts])
        assert torch.equal(many, few), how
        for r in range(10):
            n = int(counts[r])
            assert many[r].tolist() == sample_row(x[r, :n].float().numpy().astype(np.float64), u[r].numpy().astype(np.float64), **how), (r, how)
    for k in (1, m, 60, 120, 256):
        many = L.top_rows(dx, k, counts=dc, temperature=t)
        few = [L.top_rows(dx[s], k, counts=dc[s].contiguous(), temperature=t) for s in parts]
        assert torch.equal(many.index, torch.cat([f.index for f in few])) and torch.equal(many.values, torch.cat([f.values for f in few]))
        # (sums of 32 places a lane, or 2 a thread, and a tree: 64 half steps of the sum at most, and a logarithm's)
        a, b = many.lse, torch.cat([f.lse for f in few])
        assert torch.equal(a.isinf(), b.isinf())
        both = a.isfinite()
        assert ((a[both] - b[both]).abs() <= 2.0 ** -24 * (4 * b[both].abs() + 80)).all()
    y = make_logits(rows, width, dtype, seed=width + 1)
    v, i, s = make_teacher(y, m, t, 4, counts, True)
    check_distill(y, v, i, s, t, counts)
    check_distill(y, v, i, None, t, counts, torch.rand(rows, generator=rng(8)))


@pytest.mark.parametrize("width", [1500, 8200, 40000])
@pytest.mark.parametrize("ties", [False, True])
def test_sample_wide_rows_every_way(width, ties):
    """The list, the histogram, and the general form that takes what overflows them."""
    x = make_logits(3, width, F32, seed=width, ties=ties)
    u = torch.rand(3, 3, generator=rng(7))
    for how in (dict(top_k=1), dict(top_k=200), dict(top_k=512, top_p=0.9), dict(top_k=513), dict(top_k=1400, min_p=0.01, top_p=0.8),
                dict(top_p=0.3), dict(top_p=0.99, min_p=0.001), dict(top_p=0.9, temperature=0.05), dict(top_p=0.6, temperature=40.0),
                dict(top_p=0.5, temperature=1e-30), dict(temperature=1e30, top_p=0.5), dict(min_p=0.5), dict(temperature=0.0)):
        check_sample(x, u, **how)
    counts = torch.tensor([width, 700, 1], dtype=torch.int32)
    check_sample(x, u, counts=counts, top_p=0.9)
    check_sample(x, u, counts=counts, top_k=100)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width,off,ld", [(64, 0, 64), (64, 1, 70), (63, 3, 67), (250, 8, 264), (500, 5, 511), (1000, 16, 1024),
                                          (1500, 7, 1511)])
def test_strides_and_offsets(dtype, width, off, ld):
    rows = 9
    whole = make_logits(rows, ld + off, dtype, seed=ld).to(DEV)
    whole[:, :off] = 1000.0
    whole[:, off + width:] = 1000.0            # what lies beside the rows is never read as theirs
    x = whole[:, off:off + width]
    dense = x.cpu().contiguous()
    u = torch.rand(rows, 2, generator=rng(4))
    got = L.sample_rows(x, u.to(DEV), top_p=0.9).cpu()
    assert torch.equal(got, L.sample_rows(dense.to(DEV), u.to(DEV), top_p=0.9).cpu())
    check_sample(dense, u, top_p=0.9)
    top, ref = L.top_rows(x, 5), L.top_rows(dense.to(DEV), 5)
    assert all(torch.equal(a, b) for a, b in zip(top[:3], ref[:3]))
    if width <= 1024:
        (l0, g0), (l1, g1) = (L.distill_loss_and_grad(v, ref) for v in (x, dense.to(DEV)))
        assert torch.equal(l0, l1) and torch.equal(g0, g1)
    else:      # (a wide row's sums are taken in an order that its alignment shapes: against 64 bits, not bit for bit)
        v, i, s = make_teacher(dense, 5, 1.0, 3, None, True)
        check_distill(x, v, i, s, 1.0)
    same = dense[:1].to(DEV).expand(rows, width)      # one row seen many times
    assert torch.equal(L.top_rows(same, 5).index, L.top_rows(same.contiguous(), 5).index)


@pytest.mark.parametrize("width", [1, 5, 16, 64, 65, 256, 300, 512, 1000, 1024, 1025, 9000, 20001])
def test_top(width):
    rows = 23 if width <= 1024 else 5
    for i, (m, t) in enumerate(((1, 1.0), (4, 2.0), (16, 0.7), (64, 1.0), (256, 3.0))):
        dtype = (F32, F16, BF16)[(i + width) % 3]
        x = make_logits(rows, width, dtype, seed=width * 7 + i, ties=i % 2 == 0)
        if rows > 8:
            x[3] = -math.inf
            x[4, ::2] = float("nan")
            x[5] = torch.finfo(dtype).min
            x[6, ::2] = -math.inf
            x[7] = 2.0
            x[8, ::2] = -0.0
        counts = make_counts(rows, width, i) if i % 2 else None
        got = L.top_rows(x.to(DEV), m, counts=None if counts is None else counts.to(DEV), temperature=t)
        xs = x.float().numpy().astype(np.float64)
        for r in range(rows):
            n = width if counts is None else int(counts[r])
            v, at, lse = top_row(xs[r, :n], m, float(np.float32(t)))
            assert np.array_equal(got.index[r].cpu().numpy(), at), (r, m, n)
            assert np.array_equal(got.values[r].cpu().numpy().astype(np.float64), v)
            g = float(got.lse[r])
            if abs(lse) > 3.4028235e38:      # outside the range of 32 bits (the type's lowest value over t < 1): rounds to infinity
                assert g == math.copysign(math.inf, lse)
            else:      # 32 bits: sums of up to width/1024 numbers a thread and a tree over them, an exponential and a log
                y = np.abs(xs[r, :n][np.isfinite(xs[r, :n])] / t).max()
                assert abs(g - lse) <= 2.0 ** -24 * (4 * min(y, abs(lse) + 200) + 4 * abs(lse) + 64 + width / 1024), (g, lse)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [16, 33, 64, 130, 256, 400, 512, 900, 1024])
def test_top_of_rows_whose_places_do_not_part(width, dtype):
    """Equal and infinite logits, masks of the lowest value, fewer places than are asked for, for every length of the list."""
    inf = float("inf")
    x = make_logits(12, width, F32, seed=width)
    x[0] = 2.5
    x[1] = inf
    x[2, ::2] = inf
    x[3, 5:] = torch.finfo(dtype).min
    x[4, 3:] = -inf
    x[5] = torch.randint(0, 2, (width,), generator=rng(1)).float()
    x[6] = -inf
    x[7, : width // 2] = x[7].max()
    x[8] = torch.where(torch.rand(width, generator=rng(2)) < 0.5, -inf, 1.0)
    x[9, 1:] = 1e-3 * x[9, 1:]
    x[9, 0] = 1e6
    x[10] = torch.linspace(1.0, 1.0 + 2.0 ** -20, width)
    x[11] = torch.finfo(dtype).min
    x = x.to(dtype)
    y = x.float().numpy().astype(np.float64)
    for m in (1, 5, 8, 9, 16, 17, 32, 33, 48, 49, 64, 65, 96, 97, 128, 129, 200, 256):
        top = L.top_rows(x.to(DEV), m, temperature=1.0)
        values, index = top.values.cpu().numpy(), top.index.cpu().numpy()
        for r in range(12):
            v, i, _ = top_row(y[r], m, 1.0)
            assert np.array_equal(index[r], i), (m, r)
            assert np.array_equal(values[r].astype(np.float64), v), (m, r)


def make_teacher(x, m, t, seed, counts, tail):
    """A teacher near the student: its top m in 64 bits, as stored in 32."""
    rows, width = x.shape
    y = x.float() + 0.7 * torch.randn(rows, width, generator=rng(seed + 5))
    v, i, s = torch.empty(rows, m), torch.empty(rows, m, dtype=torch.int32), torch.empty(rows)
    for r in range(rows):
        n = width if counts is None else int(counts[r])
        a, b, c = top_row(y[r, :n].numpy().astype(np.float64), m, t)
        v[r], i[r], s[r] = torch.from_numpy(a), torch.from_numpy(b), c
    return v, i, s if tail else None


def check_distill(x, v, i, s, t, counts=None, weight=None):
    d = lambda a: None if a is None else a.to(DEV)
    kw = dict(counts=d(counts), weight=d(weight), temperature=t, tail=s is not None)
    top = L.TopRows(d(v), d(i), d(s))
    loss, grad = L.distill_loss_and_grad(d(x), top, **kw)
    leaf = d(x).detach().requires_grad_(True)
    up = torch.randn(x.size(0), generator=rng(9))
    alone = L.distill_loss(leaf, top, reduction="none", **kw)
    alone.backward(up.to(DEV))
    assert torch.equal(alone.detach(), loss) or torch.isnan(loss).any()
    step, xs, t64 = HALF_STEP[x.dtype], x.detach().cpu().float().numpy().astype(np.float64), float(np.float32(t))
    tiny = 2.0 ** -25 if x.dtype == F16 else 2.0 ** -134      # half of the smallest step near zero
    for r in range(x.size(0)):
        n = x.size(1) if counts is None else int(counts[r])
        w = 1.0 if weight is None else float(weight[r])
        l, g, le, ge = distill_row(xs[r, :n], v[r].numpy().astype(np.float64), i[r].numpy(), None if s is None else float(s[r]), t64, w)
        assert abs(float(loss[r]) - l) <= le + 2.0 ** -24 * abs(l), (r, n, float(loss[r]), l, le)
        got, own = grad[r].float().cpu().numpy().astype(np.float64), leaf.grad[r].float().cpu().numpy().astype(np.float64)
        assert np.all(got[n:] == 0) and np.all(own[n:] == 0)
        assert np.all(np.abs(got[:n] - g) <= ge * (1 + 2 * step) + (step + 2.0 ** -22) * np.abs(g) + tiny), (r, n)
        f = float(up[r])
        assert np.all(np.abs(own[:n] - f * g) <= abs(f) * ge * (1 + 2 * step) + (step + 2.0 ** -22) * np.abs(f * g) + tiny), (r, n)
    return loss, grad


@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("width", [1, 3, 16, 64, 65, 256, 300, 512, 777, 1024, 1025, 9000])
def test_distill(width, tail):
    rows = 21 if width <= 1024 else 4
    for k, (m, t) in enumerate(((1, 1.0), (4, 2.0), (16, 0.6), (60, 1.5), (256, 4.0))):
        dtype = (F32, BF16, F16)[(k + width) % 3]
        x = make_logits(rows, width, dtype, seed=width + 31 * k)
        counts = make_counts(rows, width, k) if k % 2 else None
        v, i, s = make_teacher(x, m, t, k, counts, tail)
        check_distill(x, v, i, s, t, counts, torch.rand(rows, generator=rng(k)) if k % 3 == 0 else None)


@pytest.mark.parametrize("width", [48, 300, 2000])
def test_distill_special_rows(width):
    t, m, rows = 1.25, 6, 12
    x = make_logits(rows, width, F32, seed=width)
    v, i, s = make_teacher(x, m, t, 3, None, True)
    i[0] = -1                                  # no entry: nothing to learn
    v[1, 2:] = -math.inf                       # entries that are absent by their logit
    i[2, 1:] = i[2, 0]                         # one place named by every entry
    i[3, 3] = width + 5                        # a place that the student's row does not have
    i[3, 4] = -7
    x[4] = -math.inf                           # a student without a place
    x[5, 1::2] = -math.inf                     # masked places of the student
    i[5] = torch.tensor([0, 2, 4, 6, 8, 10])
    x[6, 20:] = -1000.0                        # what is not listed is out of reach of 32-bit exponentials
    i[6], v[6], s[6] = torch.arange(6), x[6, :6], torch.logsumexp(x[6, :20].double() / t, 0).float() + 0.5
    x[6, 6:20] = -1100.0
    x[7] = torch.finfo(F32).min
    x[7, 0] = 0.0
    i[7] = torch.tensor([0, 1, 2, 3, 4, 5])
    v[7] = torch.tensor([0.0, -1, -2, -3, -4, -5]) 
    s[7] = float(torch.logsumexp(v[7].double() / t, 0))
    x[7, :6] = torch.tensor([0.0, -2, -1, -3, -5, -4])
    weight = torch.rand(rows, generator=rng(2))
    weight[8] = 0.0
    loss, grad = check_distill(x, v, i, s, t, None, weight)
    assert float(loss[0]) == 0 and float(loss[4]) == 0 and float(loss[8]) == 0
    assert not grad[0].any() and not grad[4].any() and not grad[8].any()
    check_distill(x, v, i, None, t, None, weight)
    # a NaN or an infinity among the student's valid logits shows; past the count it does not
    x = make_logits(3, width, F32, seed=1)
    v, i, s = make_teacher(x, m, t, 4, None, True)
    bad = x.clone()
    bad[0, 3], bad[1] = float("nan"), float("nan")
    loss, grad = L.distill_loss_and_grad(bad.to(DEV), L.TopRows(v.to(DEV), i.to(DEV), s.to(DEV)), temperature=t)
    assert torch.isnan(loss[:2]).all() and torch.isnan(grad[:2, :3]).all() and torch.isfinite(loss[2]) and torch.isfinite(grad[2]).all()
    counts = torch.full((3,), width - 2, dtype=torch.int32)
    far = x.clone()
    far[:, width - 2:] = float("nan")
    v, i, s = make_teacher(x, m, t, 4, counts, True)
    check_distill(far, v, i, s, t, counts)


@pytest.mark.parametrize("width", [40, 300, 1500])
def test_distill_every_unmasked_place_listed(width):
    """The valid places that are not listed hold nothing: no rest, and their gradient is 0."""
    x = torch.full((4, width), -math.inf)
    x[:, ::9] = torch.randn(4, (width + 8) // 9, generator=rng(2))
    m = min((width + 8) // 9, 256)
    x[:, 9 * m:] = -math.inf
    index = (torch.arange(m, dtype=torch.int32) * 9).expand(4, m).contiguous()
    values = torch.randn(4, m, generator=rng(3))
    lse = torch.logsumexp(values.double(), 1).float() + 0.25         # the teacher has something left that the student cannot reach
    loss, grad = check_distill(x, values, index, lse, 1.0)
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all() and not grad[:, 1::9].any()


@pytest.mark.parametrize("width", [5, 48, 200, 500, 1000, 1500])
def test_distill_one_place_named_many_times(width):
    """Entries that repeat a place add up to more than a row's probability.  (The bounds hold: entries of q each, added in
    steps of 2^-23, are off by 2^-24 each; 16 half steps of their sum are more than that from a q of 1/16.)"""
    x = make_logits(6, width, F32, seed=width)
    for m in (4, 5, 8, 256):
        i = torch.full((6, m), 3, dtype=torch.int32)
        i[1, -1] = 1
        i[2, ::2] = 0
        v = torch.full((6, m), 1.5)
        v[3] -= 0.25 * torch.rand(m, generator=rng(m))
        v[4, 1:] = -3.0
        s = torch.full((6,), 1.5)
        s[5] = 1.0                               # (a log-sum-exp below the entries: probabilities stay at 1)
        check_distill(x, v, i, s, 1.0)
        check_distill(x, v, i, None, 1.0)


def test_distill_listed_everywhere_has_no_rest():
    x = make_logits(7, 8, F32, seed=2)
    v, i, s = make_teacher(x, 8, 1.0, 1, None, True)
    loss, grad = check_distill(x, v, i, s, 1.0)
    v2, i2, _ = make_teacher(x, 8, 1.0, 1, None, False)
    plain, _ = check_distill(x, v2, i2, None, 1.0)
    assert torch.allclose(loss, plain, atol=1e-5)


def test_distill_gradient_is_the_slope_of_the_loss():
    """Against differences of the loss in 64 bits: central, their own error about h^2."""
    width, m, t, h = 24, 5, 1.4, 1e-4
    x = make_logits(3, width, F32, seed=12)
    v, i, s = make_teacher(x, m, t, 2, None, True)
    for lse in (s, None):
        _, grad = L.distill_loss_and_grad(x.to(DEV), L.TopRows(v.to(DEV), i.to(DEV), None if lse is None else lse.to(DEV)),
                                          temperature=t, tail=lse is not None)
        for r in range(3):
            for at in range(width):
                side = []
                for e in (h, -h):
                    y = x[r].numpy().astype(np.float64)
                    y[at] += e
                    side.append(distill_row(y, v[r].numpy().astype(np.float64), i[r].numpy(), None if lse is None else float(lse[r]),
                                            float(np.float32(t)))[0])
                slope = (side[0] - side[1]) / (2 * h)
                assert abs(float(grad[r, at]) - slope) <= 1e-6 + 1e-5 * abs(slope)


def test_reductions_and_autograd_through_a_product():
    rows, width = 20000, 40
    x = make_logits(rows, width, F32, seed=21).to(DEV)
    teacher = (x + torch.randn(rows, width, generator=rng(3)).to(DEV))
    top = L.top_rows(teacher, 8, temperature=2.0)
    each = L.distill_loss(x, top, temperature=2.0, reduction="none")
    total, mean = (L.distill_loss(x, top, temperature=2.0, reduction=k) for k in ("sum", "mean"))
    want = each.double().sum()
    assert abs(float(total) - float(want)) <= 2.0 ** -23 * float(want)
    assert abs(float(mean) - float(want) / rows) <= 2.0 ** -22 * float(want) / rows
    leaf = x.clone().requires_grad_(True)
    (3.0 * L.distill_loss(leaf * 0.5, top, temperature=2.0, reduction="mean")).backward()
    _, g = L.distill_loss_and_grad(x * 0.5, top, temperature=2.0)
    assert torch.allclose(leaf.grad, g * (1.5 / rows), rtol=1e-5, atol=1e-12)
    half = L.TopRows(top.values.bfloat16(), top.index, top.lse)           # a teacher kept in half precision
    assert torch.isfinite(L.distill_loss(x, half, temperature=2.0))


# ------------------------------------------------------------------ scores by class
def make_windows(rows, width, nodes, kinds, classes, seed, counts=True):
    g = rng(seed)
    i32 = torch.int32
    cand = torch.randint(0, nodes, (rows, width), generator=g, dtype=i32)
    c = make_counts(rows, width, seed) if counts else None
    cls = torch.randint(0, classes, (nodes,), generator=g, dtype=i32)
    kind = torch.randint(0, kinds, (rows,), generator=g, dtype=i32)
    return cand, c, cls, kind


@pytest.mark.parametrize("rows,width,kinds,classes", [(1, 1, 1, 1), (7, 3, 2, 5), (300, 64, 9, 9), (500, 100, 99, 9), (129, 257, 3, 40),
                                                      (200, 512, 40, 129), (64, 700, 300, 600), (50, 1024, 7, 1024), (1000, 16, 1, 2),
                                                      (70, 1500, 4, 33)])
@pytest.mark.parametrize("ragged", [True, False])
def test_class_scores(rows, width, kinds, classes, ragged):
    cand, counts, cls, kind = make_windows(rows, width, 333, kinds, classes, seed=rows + width, counts=ragged)
    dev = [None if v is None else v.to(DEV) for v in (cand, counts, cls, kind)]
    w = L.ScoreWindows.of(*dev, kinds)
    table = torch.randn(kinds, classes, generator=rng(4)).to(DEV).requires_grad_(True)
    out = L.class_scores(table, w)
    ok = torch.ones(rows, width, dtype=torch.bool) if counts is None else torch.arange(width) < counts[:, None]
    want = table.detach().cpu()[kind.long()[:, None], cls[cand.long()].long()]
    assert torch.equal(out.detach().cpu(), want.masked_fill(~ok, -math.inf))
    g = torch.randn(rows, width, generator=rng(5))
    g[~ok] = float("nan")                      # the gradient of what is not there is not read as a value
    out.backward(g.to(DEV))
    g64 = g.double().numpy()
    g64[~ok.numpy()] = 0.0
    pair = (kind.long()[:, None] * classes + cls[cand.long()].long()).numpy().reshape(-1)
    ref = np.bincount(pair, weights=g64.reshape(-1), minlength=kinds * classes).reshape(kinds, classes)
    size = np.bincount(pair, weights=np.abs(g64).reshape(-1), minlength=kinds * classes).reshape(kinds, classes)
    # a column of a block adds at most 64 rows times its share of a row in 32 bits, everything behind that is 64 bits wide
    adds = 64 * max(1, math.ceil(width / 32))
    assert np.all(np.abs(table.grad.cpu().numpy() - ref) <= 2.0 ** -24 * (np.abs(ref) + adds * size))
    again = L.class_scores_grad(g.to(DEV), w, kinds, classes)
    assert torch.equal(again, table.grad)


def test_class_scores_ids_outside_their_range():
    cand, counts, cls, kind = make_windows(40, 30, 50, 3, 4, seed=1)
    cand[3, 4], cand[3, 5], cls[7], cls[8], kind[6], kind[9] = -1, 50, 4, -3, 3, -1
    w = L.ScoreWindows.of(*(v.to(DEV) for v in (cand, counts, cls, kind)), 3)
    table = torch.randn(3, 4, generator=rng(2)).to(DEV)
    out = L.class_scores(table, w).cpu()
    g = torch.randn(40, 30, generator=rng(3))
    grad = L.class_scores_grad(g.to(DEV), w, 3, 4).cpu()
    ref = np.zeros((3, 4))
    for r in range(40):
        for i in range(30):
            c = int(cand[r, i])
            k = int(cls[c]) if 0 <= c < 50 else -1
            if i < int(counts[r]) and 0 <= k < 4 and 0 <= int(kind[r]) < 3:
                ref[int(kind[r]), k] += float(g[r, i])
                assert float(out[r, i]) == float(table[int(kind[r]), k])
            else:
                assert float(out[r, i]) == -math.inf
    assert np.abs(grad.numpy() - ref).max() < 1e-4


# ------------------------------------------------------------------ together, streams, recordings, sizes
def test_together_a_table_learns_its_teacher():
    """The four as they are used: a teacher's scores by class, its top logits, a student's loss, the table's gradient -
    against the same chain in 64 bits - and fan-ins drawn from the student."""
    rows, width, kinds, classes, t = 2000, 48, 9, 9, 2.0
    cand, counts, cls, kind = make_windows(rows, width, 700, kinds, classes, seed=11)
    w = L.ScoreWindows.of(*(v.to(DEV) for v in (cand, counts, cls, kind)), kinds)
    teacher = torch.randn(kinds, classes, generator=rng(6)).to(DEV)
    student = torch.randn(kinds, classes, generator=rng(7)).to(DEV).requires_grad_(True)
    top = L.top_rows(L.class_scores(teacher, w), 8, counts=w.counts, temperature=t)
    logits = L.class_scores(student, w)
    loss = L.distill_loss(logits, top, counts=w.counts, temperature=t, reduction="mean")
    loss.backward()
    ref = student.detach().double().cpu().requires_grad_(True)
    ok = torch.arange(width) < counts[:, None]
    x = ref[kind.long()[:, None], cls[cand.long()].long()].masked_fill(~ok, -1e300)
    y = teacher.double().cpu()[kind.long()[:, None], cls[cand.long()].long()].masked_fill(~ok, -math.inf)
    at = top.index.cpu().long()
    has = at >= 0
    q = torch.softmax(y / t, dim=1).nan_to_num(0.0).gather(1, at.clamp(min=0)) * has
    logp = torch.log_softmax(x / t, dim=1)
    each = (torch.where(q > 0, q * (torch.log(q.clamp(min=1e-300)) - logp.gather(1, at.clamp(min=0))), torch.zeros_like(q))).sum(1)
    mask = torch.zeros(rows, width + 1, dtype=torch.bool).scatter_(1, torch.where(has, at, width), True)[:, :width]
    rest_p = (torch.exp(logp) * (~mask & ok)).sum(1)
    use = (~mask & ok).any(1) & (counts > 0)
    rest_q = (1 - q.sum(1)).clamp(min=0)
    each = each + torch.where(use, rest_q * (torch.log(rest_q.clamp(min=1e-300)) - torch.log(rest_p.clamp(min=1e-300))), torch.zeros_like(each))
    want = (t * t * each * (counts > 0)).mean()
    want.backward()
    assert abs(float(loss) - float(want)) <= 1e-5 * abs(float(want))
    assert (student.grad.cpu().double() - ref.grad).norm() <= 1e-5 * ref.grad.norm()
    picks = L.sample_rows(logits.detach(), torch.rand(rows, 2, generator=rng(8)).to(DEV), counts=w.counts, top_p=0.9)
    assert ((picks >= 0).sum(1).cpu() <= counts).all() and (picks.cpu() < counts[:, None].clamp(min=1)).all()
    assert (picks[:, 0] != picks[:, 1])[picks[:, 1] >= 0].all()


@pytest.mark.parametrize("width", [64, 300, 5000])
def test_on_another_stream_and_recorded(width):
    rows = 200
    x = make_logits(rows, width, F32, seed=width).to(DEV)
    u = torch.rand(rows, 2, generator=rng(1)).to(DEV)
    teacher = x + torch.randn(rows, width, generator=rng(2)).to(DEV)
    cand, counts, cls, kind = make_windows(rows, width, 100, 5, 9, seed=2, counts=False)
    w = L.ScoreWindows.of(cand.to(DEV), None, cls.to(DEV), kind.to(DEV), 5)

    def everything():
        top = L.top_rows(teacher, 8)
        loss, grad = L.distill_loss_and_grad(x, top)
        return (L.sample_rows(x, u, top_k=20, top_p=0.9), *top[:3], loss, grad, L.distill_loss(x, top),
                L.class_scores_grad(grad, w, 5, 9), L.class_scores(x[:5, :9].contiguous(), w))

    want = [v.clone() for v in everything()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = everything()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        held = everything()
    for k in range(4):
        x.copy_(make_logits(rows, width, F32, seed=100 + k))
        u.copy_(torch.rand(rows, 2, generator=rng(50 + k)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in held]
        want = everything()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_an_autograd_graph_is_not_recorded():
    x = make_logits(8, 20, F32, seed=1).to(DEV).requires_grad_(True)
    top = L.top_rows(x, 4)
    cand, counts, cls, kind = make_windows(8, 20, 30, 2, 3, seed=2, counts=False)
    w = L.ScoreWindows.of(cand.to(DEV), None, cls.to(DEV), kind.to(DEV), 2)
    table = torch.zeros(2, 3, device=DEV, requires_grad=True)
    alive = L.distill_loss(x, top), L.class_scores(table, w)         # an eager graph of the same leaves
    want = L.distill_loss_and_grad(x, top)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        for call in (lambda: L.distill_loss(x, top), lambda: L.class_scores(table, w)):
            with pytest.raises(_abi.AigAbiError, match="not recorded"):
                call()
        held = L.distill_loss_and_grad(x, top)
    for _ in range(3):
        for v in held:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    alive[0].backward()
    assert x.grad is not None
    loss = L.distill_loss(x, top)
    with pytest.raises(RuntimeError, match="once"):
        loss.backward(create_graph=True)


def test_rows_far_apart():
    """Rows whose offsets pass 32 bits."""
    ld, width = 2 ** 31 + 1000, 2000
    try:
        whole = torch.empty(ld + width, dtype=F16, device=DEV)
    except torch.OutOfMemoryError:
        pytest.skip("needs 4.3 GB of device memory")
    for w in (50, width):
        x = whole.as_strided((2, w), (ld, 1))
        x.copy_(make_logits(2, w, F16, seed=w))
        dense = x.contiguous()
        u = torch.rand(2, 2, generator=rng(3)).to(DEV)
        assert torch.equal(L.sample_rows(x, u), L.sample_rows(dense, u))
        top = L.top_rows(dense, 4)
        assert all(torch.equal(a, b) for a, b in zip(L.top_rows(x, 4)[:3], top[:3]))
        assert all(torch.equal(a, b) for a, b in zip(L.distill_loss_and_grad(x, top), L.distill_loss_and_grad(dense, top)))


def test_widest_rows_and_no_rows():
    x = make_logits(2, L.MAX_WIDTH, BF16, seed=1)
    u = torch.rand(2, 2, generator=rng(1))
    check_sample(x, u, top_p=0.9)
    check_sample(x, u, top_k=300)
    check_sample(torch.zeros(1, L.MAX_WIDTH), u[:1], top_p=0.5)         # one value throughout
    v, i, s = make_teacher(x, 200, 1.0, 1, None, True)
    check_distill(x, v, i, s, 1.0)
    none = torch.empty(0, 10, device=DEV)
    assert L.sample_rows(none, torch.empty(0, 2, device=DEV)).shape == (0, 2)
    top = L.top_rows(none, 3)
    assert top.values.shape == (0, 3) and L.distill_loss_and_grad(none, top)[1].shape == (0, 10)
    assert float(L.distill_loss(none, top, reduction="sum")) == 0.0


def test_refused_on_the_device():
    x = torch.zeros(4, 8, device=DEV)
    u = torch.zeros(4, 2, device=DEV)
    top = L.top_rows(x, 2)
    bad = _abi.AigAbiError
    for call, error in (
            (lambda: L.sample_rows(x.double(), u), bad), (lambda: L.sample_rows(x.t().contiguous().t(), u), bad),
            (lambda: L.sample_rows(x[0], u), bad), (lambda: L.sample_rows(x, u[:3]), bad), (lambda: L.sample_rows(x, u.double()), bad),
            (lambda: L.sample_rows(x, torch.zeros(4, 9, device=DEV)), bad), (lambda: L.sample_rows(x, u.cpu()), bad),
            (lambda: L.sample_rows(x, u, counts=torch.zeros(4, device=DEV)), bad),
            (lambda: L.sample_rows(x, u, counts=torch.zeros(3, dtype=torch.int32, device=DEV)), bad),
            (lambda: L.sample_rows(x, u, temperature=-1.0), ValueError), (lambda: L.sample_rows(x, u, top_p=1.5), ValueError),
            (lambda: L.sample_rows(x, u, min_p=float("nan")), ValueError), (lambda: L.sample_rows(x, u, top_k=-1), ValueError),
            (lambda: L.sample_rows(x, u, temperature=torch.ones(3, device=DEV)), bad),
            (lambda: L.sample_rows(torch.zeros(1, L.MAX_WIDTH + 1, device=DEV), u[:1]), bad),
            (lambda: L.top_rows(x, 0), ValueError), (lambda: L.top_rows(x, 257), ValueError),
            (lambda: L.top_rows(x, 2, temperature=0.0), ValueError), (lambda: L.top_rows(x, 2, temperature=1e7), ValueError),
            (lambda: L.distill_loss(x, top, temperature=2.0), ValueError),              # lse taken at another temperature
            (lambda: L.distill_loss(x, L.TopRows(top.values, top.index, None)), ValueError),
            (lambda: L.distill_loss(x, top, reduction="max"), ValueError),
            (lambda: L.distill_loss(x, L.TopRows(top.values, top.index.long(), top.lse)), bad),
            (lambda: L.distill_loss(x, L.TopRows(top.values[:3], top.index, top.lse)), bad),
            (lambda: L.distill_loss(x[:0], L.top_rows(x[:0], 2)), ValueError)):
        with pytest.raises(error):
            call()
    w = L.ScoreWindows.of(*(v.to(DEV) for v in make_windows(4, 8, 10, 2, 3, seed=1)), 2)
    table = torch.zeros(2, 3, device=DEV)
    for t, ws in ((table.half(), w), (table[:1], w), (table, w._replace(cand=w.cand.long())), (table.t().contiguous().t(), w),
                  (table, w._replace(kind_start=w.kind_start[:2])), (torch.zeros(2, 1025, device=DEV), w)):
        with pytest.raises(bad):
            L.class_scores(t, ws)
    torch.cuda.synchronize()
