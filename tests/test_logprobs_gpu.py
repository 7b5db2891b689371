"""Log-probabilities of given tokens, entropy and top alternatives, and their gradient, against plain
64-bit formulas of the same logits: every vocabulary width from one word up, odd pitches, banned
words, ties, infinities and NaN, and the gradient also against differences of the forward."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, F = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F: U}
LOWEST = {BF: torch.finfo(BF).min, F: torch.finfo(F).min}


def _k():
    from imagecaptioningconvnext_amd import kernels
    return kernels


def _logits(n, V, dtype, dev, pad=0, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, V + pad, generator=g) * spread).to(dtype).to(dev)


def _forward(x, targets):
    """(logp, entropy, log p, tolerance of both) in 64 bits of x [n, V].

    Tolerance.  y = x - m is one fp32 rounding, U |y|; exp adds U |y| for its argument's factor and
    2^-22 itself, so with a = sum p |y| the sums s and t are off by w = 2 U a + 2^-22 + (V / 64 + 64) U
    relative to sum p and sum p |y| (the products y e add U).  ln s: w, and 4 U of its own size.
    logp = y - ln s: U (|y| + |ln s| + |logp|) more; H = ln s - t / s: w + 2 w a, and 4 U (|ln s| + a)."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    y = torch.where(x == -math.inf, -math.inf, x - m)
    logq = torch.log_softmax(x, -1)
    p = logq.exp()
    ent = -torch.where(p > 0, p * logq, 0.0).sum(-1)
    live = (targets >= 0) & (targets < x.shape[1])
    at = torch.where(live, targets, 0)[:, None]
    logp = torch.where(live, logq.gather(-1, at)[:, 0], 0.0)
    a = torch.where(p > 0, p * y.abs(), 0.0).sum(-1)
    ls = (m[:, 0] - torch.logsumexp(x, -1)).abs()
    w = 2 * U * a + 2.0 ** -22 + (x.shape[1] / 64 + 64) * U
    yt = torch.where(live, y.gather(-1, at)[:, 0].abs(), 0.0)
    ltol = w + 4 * U * ls + U * (yt + ls + logp.abs())
    etol = w + 2 * w * a + 4 * U * (ls + a)
    return logp, ent, logq, ltol, etol


def _order(x, top):
    """Alternatives of rows x: larger first, equal ones by index, NaN last."""
    key = torch.where(torch.isnan(x), -math.inf, x.double())
    nan = torch.isnan(x)
    ids = torch.arange(x.shape[1]).expand(x.shape)
    rows = [sorted(range(x.shape[1]), key=lambda i: (n[i], -k[i], i))[:top] for k, n in zip(key.tolist(), nan.tolist())]
    return torch.tensor(rows, dtype=torch.int64).view(x.shape[0], top)


def _check(x, V, targets, top, dev):
    K = _k()
    logp, ent, stats, tl, ti = K.token_logprobs(x, targets.to(dev), V, top=top)
    xs = x[:, :V].cpu()
    want, went, logq, ltol, etol = _forward(xs, targets)
    assert logp.shape == want.shape and tl.shape == ti.shape == (x.shape[0], top)
    inf = want == -math.inf
    assert torch.equal(logp.cpu() == -math.inf, inf)
    assert bool(((logp.cpu().double() - want).abs()[~inf] <= ltol[~inf]).all())
    assert bool(((ent.cpu().double() - went).abs() <= etol).all())
    ids = _order(xs, top)
    assert torch.equal(ti.cpu(), ids)
    wl = logq.gather(-1, ids)
    fine = wl > -math.inf
    assert torch.equal(tl.cpu() > -math.inf, fine)
    room = ltol[:, None] + 4 * U * wl.abs()
    assert bool(((tl.cpu().double() - wl).abs()[fine] <= room.expand_as(wl)[fine]).all())
    return logp, ent, stats


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 100, 255, 256, 257, 2049, 4100, 9490, 12289, 16385, 24577, 33000, 50257])
def test_forward(hip_device, dtype, V):
    g = torch.Generator().manual_seed(V)
    n = 5
    targets = torch.randint(0, V, (n,), generator=g)
    targets[1] = -1
    for pad, top in ((0, min(V, 5)), (3, min(V, 64)), (8 - V % 8, 0)):
        _check(_logits(n, V, dtype, hip_device, pad, V), V, targets, top, hip_device)


@pytest.mark.parametrize("dtype,V", [(BF, 131072), (BF, 131073), (F, 65537), (F, 140000), (BF, 300001)])
def test_forward_wide(hip_device, dtype, V):
    targets = torch.tensor([V - 1, 0, V])
    _check(_logits(3, V, dtype, hip_device, 0, V), V, targets, 20, hip_device)


@pytest.mark.parametrize("dtype", [BF, F])
def test_forward_many_rows(hip_device, dtype):
    n, V = 1500, 333
    targets = torch.randint(-1, V + 1, (n,), generator=torch.Generator().manual_seed(1))
    _check(_logits(n, V, dtype, hip_device, 3, 1), V, targets, 3, hip_device)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("V", [40, 1000, 9490, 70000])
def test_forward_ties(hip_device, dtype, V):
    """Equal logits: alternatives by index; whole rows of one value among them."""
    x = torch.zeros(6, V, dtype=dtype)
    x[1] = -2.5
    x[2] = torch.arange(V) % 3
    x[3, V // 2:] = 1
    x[4] = -0.0
    x[4, V // 3] = 0.0
    x[5] = torch.randint(0, 4, (V,), generator=torch.Generator().manual_seed(2))
    _check(x.to(hip_device), V, torch.tensor([0, V - 1, 2, V // 2, V // 3, 7]), min(V, 33), hip_device)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("V", [30, 9490, 40001])
def test_forward_banned_words(hip_device, dtype, V):
    """-inf and the type's lowest value on words that must not come; targets among them too."""
    K, dev = _k(), hip_device
    x = _logits(6, V, dtype, dev, 0, 3)
    x[0, ::2] = -math.inf
    x[1, 1:] = -math.inf                  # one word left
    x[2, 5:] = LOWEST[dtype]
    x[3] = LOWEST[dtype]                  # all banned alike: all alike
    x[4, :V - 2] = -math.inf
    x[5, 3] = -LOWEST[dtype]              # the largest value beside ordinary ones
    logp, ent, stats = _check(x, V, torch.tensor([0, 0, 6, 1, V - 1, 3]), min(V, 8), dev)
    assert logp[0] == -math.inf and logp[1] == 0 and ent[1] == 0 and abs(ent[3].item() - math.log(V)) < 1e-5
    x[:] = -math.inf                      # nothing left
    logp, ent, stats, tl, ti = K.token_logprobs(x, torch.tensor([0, 1, 2, 3, -1, V], device=dev), top=3)
    assert logp.tolist() == [-math.inf] * 4 + [0, 0] and bool((ent == 0).all()) and bool((tl == -math.inf).all())
    assert ti.tolist() == [[0, 1, 2]] * 6
    d = K.token_logprobs_bwd(x, torch.zeros(6, dtype=torch.int64, device=dev), stats, ent, torch.ones(6, device=dev),
                             torch.ones(6, device=dev))
    assert bool((d[:, 1:] == 0).all()) and bool((d[:, 0] == 1).all())


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("V", [30, 9490, 70001])
def test_nan_and_infinity_reach_their_row(hip_device, dtype, V):
    K, dev = _k(), hip_device
    x = _logits(5, V, dtype, dev, 0, 4)
    t = torch.tensor([1, 2, 3, 4, 5], device=dev)
    one = torch.ones(5, device=dev)
    clean = K.token_logprobs(x, t, top=4)
    gclean = K.token_logprobs_bwd(x, t, clean[2], clean[1], one, one)
    x[1, V // 2] = math.nan
    x[2, 7] = math.inf
    x[3] = math.nan
    logp, ent, stats, tl, ti = K.token_logprobs(x, t, top=4)
    for r in (1, 2, 3):
        assert math.isnan(logp[r]) and math.isnan(ent[r]) and bool(torch.isnan(tl[r]).all())
    assert torch.equal(ti.cpu(), _order(x.cpu(), 4))
    d = K.token_logprobs_bwd(x, t, stats, ent, one, one)
    assert bool(torch.isnan(d[1:4]).all())
    for a, b in zip((logp, ent, stats, tl, ti, d), (*clean, gclean)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[4], b[4])


def test_without_targets(hip_device):
    K = _k()
    x = _logits(4, 500, BF, hip_device)
    a = K.token_logprobs(x, None, top=5)
    b = K.token_logprobs(x, torch.zeros(4, dtype=torch.int64, device=hip_device), top=5)
    assert a[0] is None and all(torch.equal(p, q) for p, q in zip(a[1:], b[1:]))
    assert K.token_logprobs(x[:0], None, top=5)[3].shape == (0, 5)


def _grad(x, targets, g, h):
    """(gradient, tolerance before its rounding) in 64 bits.

    p is off by w = 2 U (|ln p| + |ln s|) + 2^-22 + its share of the sums' error (as in _forward),
    the bracket -g - h H - h ln p by 4 U of its terms' sizes and by h times the entropy's error."""
    x = x.double()
    V = x.shape[1]
    logq = torch.log_softmax(x, -1)
    p = logq.exp()
    ly = torch.where(p > 0, logq, 0.0)
    H = -(p * ly).sum(-1, keepdim=True)
    live = (targets >= 0) & (targets < V)
    g = torch.where(live, g.double(), 0.0)[:, None]
    h = h.double()[:, None]
    hit = torch.zeros_like(p).scatter_(-1, torch.where(live, targets, 0)[:, None], 1.0) * live[:, None]
    d = g * (hit - p) - h * p * (ly + H)
    m = x.amax(-1, keepdim=True)
    ls = (torch.logsumexp(x, -1, keepdim=True) - m).abs()
    a = torch.where(p > 0, p * (x - m).abs(), 0.0).sum(-1, keepdim=True)
    w0 = 2 * U * a + 2.0 ** -22 + (V / 64 + 64) * U
    w = 2 * w0 + 4 * U * (ly.abs() + 2 * ls + 1)
    size = g.abs() + h.abs() * (H + ly.abs())
    tol = p * (size * (w + 8 * U) + h.abs() * (w0 * (1 + 2 * a) + 4 * U * (ls + a))) + 4 * U * (hit * g.abs())
    return d, tol + 1e-38


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("V", [1, 2, 7, 100, 257, 4100, 9490, 33001, 140001])
@pytest.mark.parametrize("which", ["both", "logp", "entropy"])
def test_gradient(hip_device, dtype, V, which):
    K, dev = _k(), hip_device
    n = 4
    gen = torch.Generator().manual_seed(V)
    targets = torch.randint(0, V, (n,), generator=gen)
    targets[2] = -1
    g, h = torch.randn(n, generator=gen), torch.randn(n, generator=gen)
    for pad in (0, 5):
        x = _logits(n, V, dtype, dev, pad, V + 1)
        if V > 50:
            x[1, 10:30] = -math.inf
            x[0, 11] = LOWEST[dtype]
            targets[1] = 20  # a banned target: p 0, its own gradient g
        t = targets.to(dev)
        _, ent, stats, _, _ = K.token_logprobs(x, t, V)
        dl, de = (g.to(dev) if which != "entropy" else None), (h.to(dev) if which != "logp" else None)
        want, tol = _grad(x[:, :V].cpu(), targets, g if dl is not None else 0 * g, h if de is not None else 0 * h)
        got = K.token_logprobs_bwd(x, t, stats, ent, dl, de, V=V)
        assert got.shape == (n, V) and got.dtype == dtype
        off = (got.cpu().double() - want).abs()
        assert bool((off <= tol + HALF[dtype] * want.abs() + (2.0 ** -134 if dtype == BF else 0)).all()), V
        into = torch.full((n, V + 3), 5.0, device=dev, dtype=dtype)
        K.token_logprobs_bwd(x, t, stats, ent, dl, de, V=V, dlogits=into)
        assert torch.equal(into[:, :V], got) and bool((into[:, V:] == 5).all())
        tail = x[:, V:].clone()
        K.token_logprobs_bwd(x, t, stats, ent, dl, de, V=V, dlogits=x)  # in place
        assert torch.equal(x[:, :V], got) and torch.equal(x[:, V:], tail)


def test_gradient_is_that_of_the_forward(hip_device):
    """Central differences of the fp32 forward at every logit of a small row.  With step d the
    difference is off by d^2 / 6 times the third derivative (at most 12 here: |g|, |h| <= 1 and sums of
    p (1 + |ln p|)^3 below 12 at spread 1) and by the forward's own error over d (2 * 1e-6 / d)."""
    K, dev = _k(), hip_device
    V, d = 37, 2.0 ** -5
    x = _logits(1, V, F, dev, 0, 5, 1.0)
    t = torch.tensor([11], device=dev)
    g, h = torch.tensor([0.8], device=dev), torch.tensor([-0.6], device=dev)
    _, ent, stats, _, _ = K.token_logprobs(x, t)
    got = K.token_logprobs_bwd(x, t, stats, ent, g, h)[0]
    up, down = (x + s * d * torch.eye(V, device=dev) for s in (1, -1))
    vals = []
    for rows in (up, down):
        lp, en, _, _, _ = K.token_logprobs(rows, t.expand(V).contiguous())
        vals.append(g.double() * lp.double() + h.double() * en.double())
    slope = (vals[0] - vals[1]) / (2 * d)
    assert bool(((got.double() - slope).abs() <= d * d / 6 * 12 + 2e-6 / d).all())


def test_captured_and_on_another_stream(hip_device):
    K, dev = _k(), hip_device
    x = [_logits(33, 9490, BF, dev, 6, s) for s in (6, 7)]
    t = torch.randint(0, 9490, (33,), device=dev)
    g, h = torch.randn(33, device=dev), torch.randn(33, device=dev)

    def both(a):
        out = K.token_logprobs(a, t, 9490, top=5)
        return (*out, K.token_logprobs_bwd(a, t, out[2], out[1], g, h, V=9490))

    both(x[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in x:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(both(a))
        graphs.append(gr)
    for turn in range(3):
        for a in x:
            a.copy_(torch.randn(a.shape, device=dev) * 3)
        for gr in graphs:
            gr.replay()
        for a, o in zip(x, outs):
            assert all(torch.equal(p, q) for p, q in zip(o, both(a)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = both(x[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(o, both(x[0])))


def test_refusals(hip_device):
    K, dev = _k(), hip_device
    x = _logits(4, 100, F, dev)
    t = torch.zeros(4, dtype=torch.int64, device=dev)
    for bad in (dict(logits=x.half()), dict(logits=x[0]), dict(logits=x.t()), dict(targets=t.int()), dict(targets=t[:3]),
                dict(V=101), dict(V=0), dict(top=65), dict(top=-1), dict(targets=t.cpu()), dict(V=10, top=11)):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            K.token_logprobs(**{**dict(logits=x, targets=t), **bad})
    _, e, s, _, _ = K.token_logprobs(x, t)
    ok = dict(logits=x, targets=t, stats=s, entropy=e, dlogp=e, dentropy=e)
    for bad in (dict(targets=None), dict(stats=s[:, :1]), dict(entropy=e.double()), dict(dlogp=e[:2]), dict(dentropy=e.bfloat16()),
                dict(dlogits=x.bfloat16()), dict(dlogits=x[:, :50]), dict(dlogits=x[:3]), dict(V=200), dict(stats=s.cpu()),
                dict(logits=x.t())):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            K.token_logprobs_bwd(**{**ok, **bad})
