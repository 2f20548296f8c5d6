"""sample against its definition in 64 bits: sort, filter, add up, draw.  Tokens have to be equal; a log-probability is off by half a
step of fp32, and by what the weights' rounding to multiples of 2^-43 moves the kept mass, at least 1: vocab * 2^-44."""
import numpy as np
import pytest
import torch

from packkv_amd import ops

pytestmark = pytest.mark.gpu


def _rows(x, n):
    return np.asarray(x.cpu().numpy() if torch.is_tensor(x) else [x] * n).astype(np.float32).astype(np.float64)


def _want(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    R = logits.size(0)
    x, u = logits.double().cpu().numpy(), u.double().cpu().numpy()
    t, k, p, m = (_rows(s, R) for s in (temperature, top_k, top_p, min_p))
    tok, logp = np.full(R, -1, dtype=np.int64), np.full(R, -np.inf)
    for r in range(R):
        idx = np.nonzero(x[r] > -np.inf)[0]
        if idx.size == 0:
            continue
        idx = idx[np.argsort(-(x[r, idx] + 0.0), kind="stable")]
        n = idx.size
        if not t[r] > 0:
            tok[r], logp[r] = idx[0], 0.0
            continue
        if k[r] > 0:
            n = min(n, int(k[r]))
        top = x[r, idx[0]]
        with np.errstate(invalid="ignore"):
            w = np.where(x[r, idx] == top, 1.0, np.exp((x[r, idx] - top) / t[r]))
        if p[r] < 1:
            n = min(n, max(1, int((np.concatenate(([0.0], np.cumsum(w[:n])[:-1])) < p[r] * w[:n].sum()).sum())))
        if m[r] > 0:
            n = min(n, int((w >= min(m[r], 1.0)).sum()))
        edge = np.cumsum(w[:n])
        at = min(int(np.searchsorted(edge, u[r] * edge[-1], side="right")), n - 1)
        tok[r], logp[r] = idx[at], np.log(w[at]) - np.log(edge[-1])
    return tok, logp


def _check(logits, u, **kw):
    got, lp = ops.sample(logits, u, want_logprob=True, **kw)
    want, wl = _want(logits, u, **kw)
    assert got.dtype == torch.int64 and got.shape == u.shape and lp.dtype == torch.float32
    got, lp = got.cpu().numpy(), lp.double().cpu().numpy()
    assert (got == want).all(), [(int(r), int(got[r]), int(want[r])) for r in np.nonzero(got != want)[0][:5]]
    live = want >= 0
    assert (lp[~live] == -np.inf).all()
    tol = 2.0 ** -24 * np.abs(wl[live]) + logits.size(1) * 2.0 ** -44 + 2.0 ** -50
    assert (np.abs(lp[live] - wl[live]) <= tol).all(), np.abs(lp[live] - wl[live]).max()


def _logits(cuda, R, V, dtype, seed, spread=2.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn(R, V, generator=g, device=cuda) * spread
    x.scatter_add_(1, torch.randint(0, V, (R, 8), generator=g, device=cuda), 10 * torch.rand(R, 8, generator=g, device=cuda))
    return x.to(dtype), torch.rand(R, generator=g, device=cuda)


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_k=50, top_p=0.9, temperature=0.8), dict(top_p=0.5),
            dict(top_p=0.95, temperature=1.5), dict(min_p=0.05), dict(min_p=1.0), dict(top_p=0.0), dict(temperature=0.0), dict(temperature=0.01),
            dict(top_k=900, top_p=0.99, min_p=0.001, temperature=2.0), dict(temperature=1e30), dict(temperature=1e-30)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V", [(1, 1), (2, 7), (3, 1000), (1, 8191), (5, 32003), (2, 151936), (300, 4097), (40, 120001)])
def test_sample_follows_the_definition(cuda, dtype, R, V):
    for i, kw in enumerate(SETTINGS):
        print("sample case", dtype, R, V, kw, flush=True)
        _check(*_logits(cuda, R, V, dtype, seed=100 * i + V), **kw)


@pytest.mark.parametrize("R,V", [(37, 151936), (256, 32000)])
def test_settings_of_each_row(cuda, R, V):
    logits, u = _logits(cuda, R, V, torch.bfloat16, 3)
    g = torch.Generator(device=cuda).manual_seed(4)
    a = torch.rand(4, R, generator=g, device=cuda)
    t = torch.where(a[0] < 0.1, torch.zeros_like(u), 2 * a[0])
    t[0], t[1] = -1.0, float("nan")
    k = torch.where(a[1] < 0.5, torch.zeros_like(u), 3000 * a[1] ** 4).int()
    k[2], k[3] = -5, 2 ** 31 - 1
    p = torch.where(a[2] < 0.3, torch.ones_like(u), a[2])
    p[4], p[5] = 7.0, -1.0
    m = torch.where(a[3] < 0.5, torch.zeros_like(u), 0.2 * a[3])
    m[6], m[7] = 3.0, -1.0
    _check(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)


@pytest.mark.parametrize("V", [5000, 151936])
def test_long_runs_of_equal_logits(cuda, V):
    """More tokens in the bins in question than are ordered at once: a constant row, few distinct values, uniform numbers on borders."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.123], device=cuda)
    g = torch.Generator(device=cuda).manual_seed(V)
    for x in (torch.zeros(6, V, device=cuda), torch.full((6, V), -65504.0, device=cuda), torch.full((6, V), torch.finfo(torch.float32).min, device=cuda),
              torch.randint(0, 3, (6, V), generator=g, device=cuda).float(), torch.randint(0, 2, (6, V), generator=g, device=cuda) * 2.0 ** -20 + 1.0):
        for kw in (dict(), dict(top_k=V // 2), dict(top_p=0.6), dict(top_k=V - 7, top_p=0.37, min_p=0.5), dict(min_p=0.9), dict(temperature=0.3, top_p=0.9)):
            print("equal logits", V, x[0, :3].tolist(), kw, flush=True)
            _check(x, u, **kw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [3000, 40000, 60000])
def test_masks_infinities_and_nans(cuda, dtype, V):
    logits, u = _logits(cuda, 12, V, dtype, 9)
    inf, nan = float("inf"), float("nan")
    logits[0] = -inf
    logits[1] = nan
    logits[2] = -inf
    logits[2, V - 1] = -3.0
    logits[3, ::2] = -inf
    logits[4, 1::3] = nan
    logits[5, 7] = inf
    logits[6, 9::100] = inf
    logits[7] = torch.finfo(dtype).min
    logits[8] = -0.0
    logits[8, 5::7] = 0.0
    logits[9, 0] = nan
    logits[10] = -inf
    logits[10, 3:6] = 1.0
    for kw in (dict(), dict(top_k=3), dict(top_p=0.8, temperature=0.5), dict(min_p=0.1), dict(temperature=0.0)):
        got, lp = ops.sample(logits, u, want_logprob=True, **kw)
        want, _ = _want(logits, u, **kw)
        assert (got.cpu().numpy() == want).all(), (kw, got.tolist(), want.tolist())
        assert got[0] == -1 and got[1] == -1 and got[2] == V - 1 and not bool(lp.isnan().any())


def test_a_row_gives_the_same_token_alone_and_in_any_batch(cuda):
    logits, u = _logits(cuda, 300, 50000, torch.float16, 11)
    kw = dict(top_p=0.97, temperature=1.3)
    all_t, all_p = ops.sample(logits, u, want_logprob=True, **kw)
    for n in (1, 3, 40, 127, 128, 255):
        t, lp = ops.sample(logits[:n], u[:n], want_logprob=True, **kw)
        assert torch.equal(t, all_t[:n]) and torch.equal(lp, all_p[:n])


def test_row_layouts_and_outputs(cuda):
    wide, u = _logits(cuda, 6, 10011, torch.bfloat16, 12)
    for view in (wide[:, 3:9998], wide[::2, 1:], wide.t().contiguous().t()[:, :77], wide[:1].expand(6, 10011)):
        n = view.size(0)
        want = ops.sample(view.contiguous(), u[:n], top_p=0.9)
        out = torch.full((n,), 7, dtype=torch.int64, device=cuda)
        assert ops.sample(view, u[:n], top_p=0.9, out=out) is out and torch.equal(out, want)
        assert torch.equal(ops.sample(view, torch.stack((u, u), 1)[:n, 0], top_p=0.9), want)
    assert ops.sample(wide[:0], u[:0]).shape == (0,)


def test_uniform_numbers_outside_their_range(cuda):
    logits, _ = _logits(cuda, 4, 9000, torch.float32, 13)
    u = torch.tensor([-1.0, 1.0, 5.0, float("nan")], device=cuda)
    got = ops.sample(logits, u, top_k=20)
    order = torch.argsort(logits, dim=1, descending=True, stable=True)
    assert got.tolist() == [order[0, 0].item(), order[1, 19].item(), order[2, 19].item(), order[3, 0].item()]


def test_draws_follow_the_distribution(cuda):
    """2^14 equidistant uniform numbers take a token as often as its share says, to one."""
    x = torch.randn(1, 40, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    n = 1 << 14
    u = (torch.arange(n, device=cuda) + 0.5) / n
    got = torch.bincount(ops.sample(x.expand(n, 40), u, temperature=0.9), minlength=40)
    assert (got - torch.softmax(x[0].double() / 0.9, 0) * n).abs().max().item() <= 1.0


def test_two_streams_and_a_graph(cuda):
    logits, u = _logits(cuda, 3, 151936, torch.bfloat16, 14)
    kw = dict(top_k=40, top_p=0.9)
    want = ops.sample(logits, u, **kw)
    torch.cuda.synchronize()
    outs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.sample(logits, u, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, ops.sample(logits, u, **kw)))
    for step in range(4):
        logits.copy_(_logits(cuda, 3, 151936, torch.bfloat16, 20 + step)[0])
        u.uniform_()
        for g, _ in graphs:
            g.replay()
        want = ops.sample(logits, u, **kw)
        torch.cuda.synchronize()
        assert all(torch.equal(got, want) for _, got in graphs)


def test_refusals(cuda):
    logits, u = _logits(cuda, 3, 100, torch.float16, 15)

    def bad(match, logits=logits, u=u, **kw):
        with pytest.raises(RuntimeError, match=match):
            ops.sample(logits, u, **kw)

    bad("device tensor", logits=logits[0])
    bad("device tensor", logits=logits[:, :0])
    bad("Unsupported data type", logits=logits.double())
    bad("2\\^20", logits=logits[:, :1].expand(3, (1 << 20) + 1))
    for wrong in (u[:2], u.double(), u.cpu(), u[:, None]):
        bad("u must be", u=wrong)
    for kw in (dict(temperature=-0.1), dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=2.5), dict(top_k=float("inf")), dict(top_k=1 << 31), dict(top_p=1.1), dict(top_p=-0.1),
               dict(min_p=1.5), dict(min_p=float("nan"))):
        bad("out of range", **kw)
    bad("temperature must be", temperature=u[:2])
    bad("top_k must be", top_k=u)
    bad("top_p must be", top_p=u.cpu())
    bad("out must be", out=torch.zeros(3, device=cuda))


def test_rows_further_apart_than_32_bits(cuda):
    flat = torch.empty((1 << 31) + 80000, dtype=torch.bfloat16, device=cuda)
    for V in (70000, 5000):                                # in slices, and not
        far = flat.as_strided((2, V), (1 << 31, 1), 7)
        logits, u = _logits(cuda, 2, V, torch.bfloat16, V)
        far.copy_(logits)
        for kw in (dict(top_p=0.9), dict(temperature=0.0)):
            got, want = ops.sample(far, u, want_logprob=True, **kw), ops.sample(logits, u, want_logprob=True, **kw)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_most_tokens_a_row_can_have(cuda):
    V = 1 << 20
    u = torch.tensor([0.0, 0.5, 1 - 2.0 ** -24], device=cuda)
    tok, lp = ops.sample(torch.zeros(3, V, device=cuda), u, want_logprob=True)
    assert tok.tolist() == [0, V // 2, int((1 - 2.0 ** -24) * V)] and (lp + 20 * np.log(2)).abs().max().item() < 1e-6
    _check(*_logits(cuda, 2, V, torch.float16, 21), top_p=0.8)


def test_logits_about_zero_beside_an_edge_of_the_bins(cuda):
    """A temperature and a maximum that put zero on the border of two bins, to 2^-29 of the maximum: numbers around it are far closer
    together than those that differ from the maximum."""
    f32 = np.float32
    found = []
    for i in range(4000):
        t = f32(1.25) + f32(i) * f32(2.0 ** -12)
        per = 64 * 1.4426950408889634074 / float(t)
        top = f32(512 / per)
        if abs(float(top) * per / 512 - 1) < 2.0 ** -29:
            found.append((float(t), float(top)))
    assert found
    g = torch.Generator(device=cuda).manual_seed(22)
    for t, top in found[:6]:
        x = torch.randn(3, 6000, generator=g, device=cuda) * 10.0 ** (-45 * torch.rand(3, 6000, generator=g, device=cuda) ** 0.5)
        x = torch.where(x.abs() > top, torch.zeros_like(x), x)
        x[:, 17] = top
        u = torch.tensor([0.3, 0.6, 0.9], device=cuda)
        for kw in (dict(), dict(top_k=2500), dict(top_p=0.4), dict(top_p=0.41, top_k=3400)):
            _check(x, u, temperature=t, **kw)
