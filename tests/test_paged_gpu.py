"""Paged key/value cache: the planner, the writer and the attention of one new token per request,
against plain implementations (the planner's request by request on the host, the attention's in 64
bits), at the lengths, page sizes, strides and contents where they can go wrong."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32, relative
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}
BF, F = torch.bfloat16, torch.float32


def _k():
    from imagecaptioningconvnext_amd import kernels
    return kernels


def _abi():
    from imagecaptioningconvnext_amd import _abi
    return _abi


def _desc(q, kc, width, max_len):
    """The attention's descriptor, its sizes and types only, with addresses that are not read."""
    d = _abi().PagedAttnDesc()
    d.dtype, (d.B, d.H, d.dh), (d.pages, d.page, d.Hkv, _) = _k().dt(q), q.shape, kc.shape
    d.width, d.max_len, d.scale = width, max_len, 1.0
    d.q_row, d.q_head, d.o_row, d.o_head = q.stride(0), q.stride(1), q.stride(0), q.stride(1)
    d.k_page, d.k_tok, d.k_head = d.v_page, d.v_tok, d.v_head = kc.stride()[:3]
    d.table_row = width
    d.q = d.k = d.v = d.o = d.table = d.lens = kc.data_ptr()
    return d


# ---- attention ------------------------------------------------------------------------------
def _cache(lens, page, hkv, dh, dtype, seed, dev, spare=2, garbage=float("nan")):
    """(k cache, v cache, table) whose unused places hold garbage; keys and values normal."""
    g = torch.Generator().manual_seed(seed)
    have = [(n + page - 1) // page for n in lens]
    pages = sum(have) + spare
    ids = torch.randperm(pages, generator=g).tolist()
    width = max(max(have), 1) + 1
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    kc, vc = (torch.full((pages, page, hkv, dh), garbage, dtype=dtype) for _ in range(2))
    for b, n in enumerate(lens):
        for j in range(have[b]):
            table[b, j] = i = ids.pop()
            m = min(page, n - j * page)
            kc[i, :m] = torch.randn(m, hkv, dh, generator=g).to(dtype)
            vc[i, :m] = torch.randn(m, hkv, dh, generator=g).to(dtype)
    return kc.to(dev), vc.to(dev), table.to(dev)


def _reference(q, kc, vc, table, lens, scale):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits, request by request.

    Tolerance.  A score is a sum of dh products in fp32: off by at most (dh + 1) U sum|q k| scale,
    and by 2 U |score| for its factor and its difference to the maximum; with E the largest of
    scale * sum|q k|, a weight's relative error is (dh + 4) U E + 2^-22 (exponential), twice that
    with its share of the normalising sum.  Summing n terms adds n U, the joins of parts and the
    division another 64 U.  With bf16 values a weight goes in as two bf16 pieces, 2 * 2^-8 * 2^-8 of
    it at most left out.  All of that multiplies sum(p |v|); the output's rounding is half a step."""
    pages, page, hkv, dh = kc.shape
    B, H = q.shape[:2]
    out, tol = torch.zeros(B, H, dh, dtype=torch.float64), torch.zeros(B, H, dh, dtype=torch.float64)
    lse, ltol = torch.full((B, H), -math.inf, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    kc, vc, table, q = kc.cpu(), vc.cpu(), table.cpu().long(), q.cpu().double()
    for b in range(B):
        t = torch.arange(lens[b])
        ids = table[b, t // page] if lens[b] else t
        here = (ids >= 0) & (ids < pages)
        t, ids = t[here], ids[here]
        if not len(t):
            continue
        k, v = (c[ids, t % page].double().repeat_interleave(H // hkv, 1) for c in (kc, vc))  # [n, H, dh]
        s = torch.einsum("hd,nhd->hn", q[b], k) * scale
        E = (torch.einsum("hd,nhd->hn", q[b].abs(), k.abs()) * abs(scale)).amax(-1)
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("hn,nhd->hd", p, v)
        lse[b] = torch.logsumexp(s, -1)
        w = 2 * ((dh + 4) * U * E + 2.0 ** -22) + (len(t) + 64) * U
        ltol[b] = w + 4 * U * lse[b].abs()
        w = w + (2.0 ** -15 if kc.dtype == BF else 0)
        tol[b] = w[:, None] * torch.einsum("hn,nhd->hd", p, v.abs()) + HALF[kc.dtype] * out[b].abs() + 1e-30
    return out, lse, tol, ltol


def _check(q, kc, vc, table, lens, scale=None, **kw):
    K = _k()
    dev = q.device
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    lse = torch.full(q.shape[:2], 9.0, device=dev)
    got = K.paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=dev), scale=scale, lse=lse,
                            **kw)
    out, ref_lse, tol, ltol = _reference(q, kc, vc, table, lens, sc)
    off = (got.cpu().double() - out).abs()
    assert torch.isfinite(got).all()
    assert bool((off <= tol).all()), f"off {(off / tol).max().item():.2f} times the tolerance"
    fine = torch.isfinite(ref_lse)
    assert torch.equal(torch.isfinite(lse.cpu()), fine)
    assert bool(((lse.cpu().double() - ref_lse).abs()[fine] <= ltol[fine]).all())
    return got


LENS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 300]


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("H,hkv,dh", [(8, 8, 64), (4, 2, 128), (5, 1, 64), (16, 1, 128), (40, 2, 64), (3, 3, 128)])
@pytest.mark.parametrize("page", [1, 2, 8, 16, 64, 256])
def test_attention(hip_device, dtype, H, hkv, dh, page):
    kc, vc, table = _cache(LENS, page, hkv, dh, dtype, 1, hip_device)
    q = torch.randn(len(LENS), H, dh, generator=torch.Generator().manual_seed(2)).to(dtype).to(hip_device)
    _check(q, kc, vc, table, LENS)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("lens,page", [([1], 1), ([7], 16), ([32, 0], 16), ([64, 3], 2), ([0, 0], 16), ([4099], 16),
                                       ([2500, 0, 1, 5000], 32), ([1025] * 3, 1), ([9001, 12], 1024)])
def test_attention_lengths(hip_device, dtype, lens, page):
    """One wave's length, two waves', and lengths that are split over workgroups and joined."""
    kc, vc, table = _cache(lens, page, 2, 64, dtype, 3, hip_device)
    q = torch.randn(len(lens), 6, 64, generator=torch.Generator().manual_seed(4)).to(dtype).to(hip_device)
    a = _check(q, kc, vc, table, lens)
    if max(lens):  # the host's bound changes how the work is cut, not what is computed
        b = _check(q, kc, vc, table, lens, max_len=max(lens))
        assert ((a.double() - b.double()).abs() <= 4 * HALF[dtype] * a.double().abs() + 1e-4).all()


def test_attention_stops_at_the_bound(hip_device):
    kc, vc, table = _cache([100, 700], 16, 2, 64, F, 5, hip_device)
    q = torch.randn(2, 2, 64, device=hip_device)
    got = _k().paged_attention(q, kc, vc, table, torch.tensor([100, 700], dtype=torch.int32, device=hip_device), max_len=90)
    out, _, tol, _ = _reference(q, kc, vc, table, [90, 90], 0.125)
    assert bool(((got.cpu().double() - out).abs() <= tol).all())
    # longer than the table: the table's width counts; negative: none
    wide = torch.tensor([1 << 30, -5], dtype=torch.int32, device=hip_device)
    full = table.shape[1] * 16
    kc.nan_to_num_(0.25)
    vc.nan_to_num_(0.5)
    got = _k().paged_attention(q, kc, vc, table, wide)
    out, _, tol, _ = _reference(q, kc, vc, table, [full, 0], 0.125)
    assert bool(((got.cpu().double() - out).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("page", [4, 16, 128])
def test_attention_strides(hip_device, dtype, page):
    """Head-major caches, keys and values of one buffer, queries inside a packed projection, an
    output and a table that are parts of wider ones (what surrounds them stays)."""
    K, dev = _k(), hip_device
    lens = [37, 130, 1, 0, 64]
    H, hkv, dh, B = 8, 4, 64, 5
    kc, vc, table = _cache(lens, page, hkv, dh, dtype, 6, dev)
    both = torch.stack([kc.transpose(1, 2), vc.transpose(1, 2)], 1).contiguous()  # [pages, 2, heads, page, dh]
    kh, vh = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    packed = torch.randn(B, 3 * H * dh, device=dev).to(dtype)
    q = packed[:, H * dh:2 * H * dh].view(B, H, dh)
    wide = torch.full((B, H + 1, dh + 8), 3.0, device=dev, dtype=dtype)
    tab = torch.full((B, table.shape[1] + 3), 1 << 20, device=dev, dtype=torch.int32)
    tab[:, :table.shape[1]] = table
    out = wide[:, :H, :dh]
    plain = K.paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=dev))
    _check(q, kh, vh, tab[:, :table.shape[1]], lens, out=out)
    assert torch.equal(out, plain)
    assert bool((wide[:, H] == 3).all()) and bool((wide[:, :, dh:] == 3).all())


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("page", [1, 8, 32])
def test_attention_pages_outside_the_cache(hip_device, dtype, page):
    lens = [200, 90, 33]
    kc, vc, table = _cache(lens, page, 2, 64, dtype, 7, hip_device)
    table[0, 1], table[0, 64 // page] = -1, kc.shape[0]
    table[1] = 1 << 30  # a request whose pages are all bad has no keys
    table[2, 0] = -(1 << 31)
    q = torch.randn(3, 2, 64, device=hip_device).to(dtype)
    got = _check(q, kc, vc, table, lens)
    assert bool((got[1] == 0).all())


@pytest.mark.parametrize("dtype", [BF, F])
def test_attention_infinities_and_nan(hip_device, dtype):
    """What a live key or value holds reaches its own request and kv head, and nothing else's."""
    K, dev = _k(), hip_device
    lens = [70, 70, 70, 70]
    kc, vc, table = _cache(lens, 16, 2, 64, dtype, 8, dev)
    q = torch.randn(4, 4, 64, device=dev).to(dtype)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    clean = K.paged_attention(q, kc, vc, table, n)
    kc[table[0, 2], 3, 0, 5] = math.nan          # position 35 of request 0, kv head 0
    vc[table[1, 4], 5, 1, 7] = math.inf          # position 69 of request 1, kv head 1, one column
    kc[table[2, 0], 0, 1] = -math.inf * torch.sign(q[2, 2])  # weight of q head 2: exp(-inf) = 0
    got = K.paged_attention(q, kc, vc, table, n)
    assert bool(torch.isnan(got[0, :2]).all()) and torch.equal(got[0, 2:], clean[0, 2:])
    hit = torch.zeros(4, 64, dtype=torch.bool, device=dev)
    hit[2:, 7] = True
    assert bool((got[1][hit] == math.inf).all()) and torch.equal(got[1][~hit], clean[1][~hit])
    assert bool(torch.isfinite(got[2, 2]).all()) and torch.equal(got[2, :2], clean[2, :2])
    assert torch.equal(got[3], clean[3])
    none = torch.full_like(kc, math.nan)  # every score -inf: as a request without keys
    none.copy_(-math.inf * torch.sign(q[:1, :1, :]).expand_as(none))
    lse = torch.zeros(1, 4, device=dev)
    got = K.paged_attention(q[:1, :1].expand(1, 4, 64).contiguous(), none, vc, table[:1], n[:1], lse=lse)
    assert bool((got == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("page,n", [(16, 20), (1, 20), (16, 700), (16, 3000)])
def test_attention_weightless_positions(hip_device, dtype, page, n):
    """Live positions of weight 0 (scores of -200 and of -inf) that hold the type's largest values add
    nothing; one of weight e^-72 adds its share, and an infinite value is infinity at any weight above
    0.  Scores are exact (the query is 1 in one place); taken to base 2 one of 72 is off by 4 U 104, the
    exponential by 2^-22, two bf16 pieces of a weight by 2^-16: less than 2^-15 of sum(p |v|) in all."""
    kc, vc, table = _cache([n] * 3, page, 1, 64, dtype, 40, hip_device)
    at = lambda b, t: (table[b, t // page].item(), t % page, 0)  # noqa: E731
    kc[..., 0] = torch.where(kc[..., 0].isnan(), kc[..., 0], 0)
    kc[..., 1:] = 0
    q = torch.zeros(3, 2, 64, dtype=dtype, device=hip_device)
    q[..., 0] = 1
    for b in range(3):
        for t in (3, n - 2):
            kc[at(b, t)][0] = -1600
            vc[at(b, t)] = torch.finfo(dtype).max
        kc[at(b, 7)][0] = -math.inf
        vc[at(b, 7)] = torch.finfo(dtype).max
    kc[at(1, 5)][0] = -576
    vc[at(1, 5)] = 1e31
    lens = torch.tensor([n] * 3, dtype=torch.int32, device=hip_device)
    got = _k().paged_attention(q, kc, vc, table, lens)
    t = torch.arange(n, device=hip_device)
    for b in range(3):
        k, v = (c[table[b, t // page].long(), t % page, 0].double() for c in (kc, vc))
        p = torch.softmax(k[:, 0] / 8, 0)[:, None]
        want, room = (p * v).sum(0), (p * v.abs()).sum(0)
        assert bool(((got[b].double() - want).abs() <= 2.0 ** -15 * room + HALF[dtype] * want.abs()).all()), b
    for score in (-64, -576, -680):  # weights of e^-8, e^-72 and e^-85
        kc[at(2, 5)][0] = score
        vc[at(2, 5)][0] = math.inf
        got = _k().paged_attention(q, kc, vc, table, lens)
        assert bool((got[2, :, 0] == math.inf).all()) and bool(torch.isfinite(got[2, :, 1:]).all())


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_attention_scale(hip_device, scale):
    kc, vc, table = _cache([50, 3], 16, 1, 128, F, 9, hip_device)
    _check(torch.randn(2, 2, 128, device=hip_device), kc, vc, table, [50, 3], scale=scale)


@pytest.mark.parametrize("page", [64, 1])
def test_attention_far_offsets(hip_device, page):
    """A cache of more than 2^31 elements: pages at its end are where they should be."""
    dev = hip_device
    hkv, dh = 8, 128
    pages = (1 << 31) // (page * hkv * dh) + 400
    kc, vc = (torch.zeros(pages, page, hkv, dh, dtype=BF, device=dev) for _ in range(2))
    lens, g = [100, 190], torch.Generator().manual_seed(10)
    width = (190 + page - 1) // page
    table = pages - 1 - torch.randperm(2 * width, generator=g).view(2, width).to(torch.int32).to(dev)
    table[1, 1] = 3
    K = _k()
    rows = sum(lens)
    k, v = (torch.randn(rows, hkv, dh, generator=g).to(BF).to(dev) for _ in range(2))
    pos = torch.cat([torch.arange(n) for n in lens]).to(dev)
    row = torch.repeat_interleave(torch.arange(2), torch.tensor(lens)).to(dev)
    K.paged_write(k, v, kc, vc, table[row, pos // page].long() * page + pos % page)
    q = torch.randn(2, 16, dh, generator=g).to(BF).to(dev)
    got = K.paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=dev))
    used = torch.unique(table.clamp(min=0).reshape(-1).long())
    small = torch.searchsorted(used, table.clamp(min=0).long()).to(torch.int32)
    out, _, tol, _ = _reference(q, kc[used], vc[used], small, lens, dh ** -0.5)
    assert bool(((got.cpu().double() - out).abs() <= tol).all())


@pytest.mark.parametrize("dtype,H,hkv,dh,n,parts", [
    (BF, 8, 1, 64, 140001, 274), (F, 8, 1, 64, 140001, 274),     # joined by 32 columns, past 256 parts
    (BF, 96, 1, 64, 70001, 137), (F, 96, 1, 64, 70001, 137),     # by whole rows of 64, past 128
    (BF, 256, 2, 128, 35001, 69), (F, 256, 2, 128, 35001, 69),   # by whole rows of 128, past 64
    (BF, 2, 1, 64, 600001, 987), (F, 3, 1, 128, 530003, 975),    # as many parts as there can be, or nearly
])
def test_attention_of_many_parts(hip_device, dtype, H, hkv, dh, n, parts):
    """Lengths in more parts than the join takes in one round; the second row ends in its first part and
    the third in the middle of one.  As in _reference, by products of whole matrices, but for the sums:
    a term of a part of c tokens passes c / 16 additions in its lane, 32 in its workgroup, then an eighth
    of the parts and 32 more in the join."""
    K, dev = _k(), hip_device
    g = torch.Generator(dev).manual_seed(41)
    lens, page = [n, 77, n // 2 + 5], 256
    width = (n + page - 1) // page
    kc, vc = (torch.randn(width + 1, page, hkv, dh, generator=g, device=dev).to(dtype) for _ in range(2))
    table = torch.stack([torch.randperm(width + 1, generator=g, device=dev)[:width] for _ in lens]).to(torch.int32)
    q = torch.randn(3, H, dh, generator=g, device=dev).to(dtype)
    d, need = _desc(q, kc, width, n), ctypes.c_int64(0)
    assert _abi().lib().imgcap_paged_attention_ws(ctypes.byref(d), ctypes.byref(need)) == 0
    assert need.value == 3 * H * parts * (dh + 2) * 4
    lse = torch.empty(3, H, device=dev)
    got = K.paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=dev), max_len=n, lse=lse)
    for b, m in enumerate(lens):
        t = torch.arange(m, device=dev)
        k, v = (c[table[b, t // page].long(), t % page].double().transpose(0, 1).contiguous() for c in (kc, vc))
        x = q[b].double().view(hkv, H // hkv, dh)
        s = torch.matmul(x, k.transpose(1, 2).contiguous()) * dh ** -0.5
        E = torch.matmul(x.abs(), k.abs().transpose(1, 2).contiguous()).amax(-1).view(H) * dh ** -0.5
        p = torch.softmax(s, -1)
        out, room = (torch.matmul(p, w).view(H, dh) for w in (v, v.abs()))
        w = 2 * ((dh + 4) * U * E + 2.0 ** -22) + (n / parts / 16 + parts / 8 + 64) * U
        ref = torch.logsumexp(s, -1).view(H)
        assert bool(((lse[b].double() - ref).abs() <= w + 4 * U * ref.abs()).all()), b
        tol = (w + (2.0 ** -15 if dtype == BF else 0))[:, None] * room + HALF[dtype] * out.abs()
        assert bool(((got[b].double() - out).abs() <= tol).all()), b


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("B", [1, 150, 2500])
def test_attention_widest_table(hip_device, dtype, B):
    """A table of the most positions there can be (2^31 - 65536), with ordinary requests in it: lengths of
    parts, their number and the places where they begin come near 2^31 (1024 parts, 27, 2)."""
    K, dev = _k(), hip_device
    lens = [1 + 977 * (b % 4) for b in range(B)]
    lens[0] = 2500
    kc, vc, table = _cache([4096], 1024, 2, 64, dtype, 30, dev)
    wide = torch.full((1, ((1 << 31) - 65536) // 1024), -1, dtype=torch.int32, device=dev)
    wide[:, :4] = table[:, :4]
    q = torch.randn(B, 2, 64, generator=torch.Generator().manual_seed(31)).to(dtype).to(dev)
    got = K.paged_attention(q, kc, vc, wide.expand(B, -1), torch.tensor(lens, dtype=torch.int32, device=dev))
    few = sorted({0, 1, 2, 3, B // 2, B - 2, B - 1} & set(range(B)))
    out, _, tol, _ = _reference(q[few], kc, vc, table.expand(B, -1)[few], [lens[b] for b in few], 0.125)
    assert bool(((got[few].cpu().double() - out).abs() <= tol).all())


def test_attention_of_the_longest_row(hip_device):
    """2^31 - 65541 positions on three pages that come again and again and a last one, whose last
    position alone outweighs all others, so that a part that is cut short shows.  Scores: 40 against 0, so the others weigh 2^31 e^-40 =
    5e-9 in all, beside the output's half step and the two bf16 pieces of a weight."""
    K, dev = _k(), hip_device
    width = ((1 << 31) - 65536) // 1024
    n = width * 1024 - 5
    table = (torch.arange(width, device=dev, dtype=torch.int32) % 3)[None].clone()
    table[0, -1] = 3
    g = torch.Generator().manual_seed(32)
    q = torch.randn(1, 1, 64, generator=g).to(BF).to(dev)
    kc = torch.zeros(4, 1024, 1, 64, dtype=BF, device=dev)
    vc = torch.randn(4, 1024, 1, 64, generator=g).to(BF).to(dev)
    x = q[0, 0].double()
    kc[3, (n - 1) % 1024, 0] = (320 * x / (x @ x)).to(BF)
    kc[3, n % 1024:] = float("nan")
    want = vc[3, (n - 1) % 1024, 0].double()
    got = K.paged_attention(q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device=dev))
    assert bool(((got[0, 0].double() - want).abs() <= (2.0 ** -15 + HALF[BF]) * want.abs() + 1e-7).all())


def test_attention_captured_twice_and_on_another_stream(hip_device):
    """Two captured graphs of a split length replay in turn, with eager calls between, on new inputs;
    then the same on a stream of its own."""
    K, dev = _k(), hip_device
    lens = [3000, 900]
    kc, vc, table = _cache(lens, 16, 2, 64, BF, 11, dev, garbage=0.0)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    qs = [torch.randn(2, 8, 64, device=dev).to(BF) for _ in range(2)]
    K.paged_attention(qs[0], kc, vc, table, n)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K.paged_attention(q, kc, vc, table, n))
        graphs.append(g)
    for turn in range(4):
        for q in qs:
            q.copy_(torch.randn(2, 8, 64, device=dev))
        n.copy_(torch.tensor([3000 - 700 * turn, 40 + turn], device=dev))
        for g in graphs:
            g.replay()
        for q, o in zip(qs, outs):
            assert torch.equal(o, K.paged_attention(q, kc, vc, table, n))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [K.paged_attention(q, kc, vc, table, n) for q in qs * 3]
    torch.cuda.current_stream().wait_stream(side)
    for q, o in zip(qs * 3, got):
        assert torch.equal(o, K.paged_attention(q, kc, vc, table, n))


def test_attention_refuses(hip_device):
    K, dev = _k(), hip_device
    kc, vc, table = _cache([20, 20], 16, 2, 64, BF, 12, dev)
    n = torch.tensor([20, 20], dtype=torch.int32, device=dev)
    q = torch.zeros(2, 4, 64, device=dev, dtype=BF)
    ok = dict(q=q, k_cache=kc, v_cache=vc, table=table, lens=n)
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[:1]), dict(q=q[..., :32]), dict(q=q.transpose(0, 1)[:, :, ::2]),
                dict(table=table.long()), dict(table=table[:1]), dict(table=table.t()), dict(lens=n.long()), dict(lens=n[:1]),
                dict(v_cache=vc[:1]), dict(v_cache=vc.float()), dict(k_cache=kc[:, :12]), dict(out=q.float()),
                dict(out=q[:1]), dict(max_len=(1 << 32) + 32), dict(lse=torch.zeros(2, 4, device=dev, dtype=BF)), dict(max_len=0), dict(max_len=1 << 20),
                dict(lens=n.cpu()), dict(q=q.half()), dict(k_cache=kc.flatten()[4:-4092].view(-1, 16, 2, 64)[:4])):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            K.paged_attention(**{**ok, **bad})
    assert K.paged_attention(q[:0], kc, vc, table[:0], n[:0]).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", [BF, F])
def test_attention_in_place_and_single_dims(hip_device, dtype):
    """The output may be the queries' own buffer; dimensions of one have no stride that counts."""
    K, dev = _k(), hip_device
    for lens, page in (([40, 2, 0], 8), ([700, 90, 3], 16), ([2600, 5, 64], 16)):
        kc, vc, table = _cache(lens, page, 2, 64, dtype, 24, dev)
        n = torch.tensor(lens, dtype=torch.int32, device=dev)
        q = torch.randn(3, 40, 64, device=dev).to(dtype)
        want = K.paged_attention(q, kc, vc, table, n)
        assert K.paged_attention(q, kc, vc, table, n, out=q) is q and torch.equal(q, want)
    base = torch.randn(9, 67, device=dev).to(dtype)  # rows of 67: a stride that is no whole 16 bytes
    one = base[:1, :64].as_strided((1, 1, 1, 64), (67, 67, 67, 1))
    q = base[1:2].as_strided((1, 1, 64), (67, 67, 1), 0)
    got = K.paged_attention(q, one, one, torch.zeros(1, 1, dtype=torch.int32, device=dev),
                            torch.ones(1, dtype=torch.int32, device=dev))
    assert torch.equal(got[0, 0], one[0, 0, 0])
    into = torch.zeros(1, 1, 1, 64, device=dev, dtype=dtype)
    K.paged_write(q, q, into, into.clone(), torch.zeros(1, dtype=torch.int64, device=dev))
    assert torch.equal(into[0, 0, 0], base[0, :64])


# ---- the writer -----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("n,heads,dh,page", [(1, 1, 64, 1), (64, 8, 64, 16), (333, 3, 128, 2), (1000, 5, 24, 128)])
@pytest.mark.parametrize("headmajor", [False, True])
def test_write(hip_device, dtype, n, heads, dh, page, headmajor):
    K, dev = _k(), hip_device
    g = torch.Generator().manual_seed(13)
    pages = n // page + 3
    shape = (pages, heads, page, dh) if headmajor else (pages, page, heads, dh)
    caches = [torch.randn(shape, generator=g).to(dtype).to(dev) for _ in range(2)]
    kc, vc = (c.transpose(1, 2) if headmajor else c for c in caches)
    rows = torch.randn(n, 3, heads, dh, generator=g).to(dtype).to(dev)
    k, v = rows[:, 1], rows[:, 2]
    slots = torch.randperm(pages * page, generator=g)[:n]
    bad = torch.randperm(n, generator=g)[:n // 5]
    slots[bad] = torch.tensor([-1, pages * page, -(1 << 40), 1 << 40, -1])[torch.arange(len(bad)) % 5]
    want = [c.clone().cpu() for c in (kc, vc)]
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            for w, src in zip(want, (k, v)):
                w[s // page, s % page] = src[i].cpu()
    K.paged_write(k, v, kc, vc, slots.to(dev))
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])


def test_write_refuses(hip_device):
    K, dev = _k(), hip_device
    k = torch.zeros(4, 2, 64, device=dev, dtype=BF)
    c = torch.zeros(3, 16, 2, 64, device=dev, dtype=BF)
    s = torch.zeros(4, dtype=torch.int64, device=dev)
    ok = dict(k=k, v=k, k_cache=c, v_cache=c.clone(), slots=s)
    for bad in (dict(k=k.float()), dict(k=k[:3]), dict(v=k[:, :1]), dict(slots=s.int()), dict(slots=s.cpu()), dict(k_cache=c[0]),
                dict(k_cache=c[:, :10], v_cache=c[:, :10]), dict(k=k.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(k_cache=c.float(), v_cache=c.float()), dict(k=k.half(), v=k.half(), k_cache=c.half(), v_cache=c.half())):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            K.paged_write(**{**ok, **bad})
    K.paged_write(k[:0], k[:0], c, c.clone(), s[:0])


# ---- the planner ----------------------------------------------------------------------------
def _plan_ref(past, new, table, free, count, page, tokens):
    """Request by request.  Returns the outputs and the table, stack and count after the step."""
    table, free = [list(r) for r in table], list(free)
    B, width, pool = len(past), len(table[0]), len(free)
    top = min(max(count, 0), pool)
    for b in range(B):
        if new[b] < 0:
            for j in range(min((max(past[b], 0) + page - 1) // page, width)):
                if top < pool:
                    free[top] = table[b][j]
                    top += 1
    asked = pages = 0
    left = top
    lens, starts, waits, slots, rows, positions = [], [0], [], [], [], []
    for b in range(B):
        if new[b] < 0:
            lens.append(0), waits.append(0), starts.append(len(slots))
            continue
        fits = past[b] >= 0 and past[b] + new[b] <= width * page
        if fits:
            asked += new[b]
            fits = asked <= tokens
        have = (max(past[b], 0) + page - 1) // page
        need = (past[b] + new[b] + page - 1) // page - have if fits else 0
        pages += need
        ok = fits and (need == 0 or pages <= top)
        if ok:
            for j in range(have, have + need):
                table[b][j] = free[left - 1]
                left -= 1
            for p in range(past[b], past[b] + new[b]):
                i = table[b][p // page]
                slots.append(i * page + p % page if 0 <= i < pool else -1)
                rows.append(b), positions.append(p)
        lens.append(past[b] + (new[b] if ok else 0)), waits.append(0 if ok else 1), starts.append(len(slots))
    pad = tokens - len(slots)
    return (lens, starts, slots + [-1] * pad, rows + [-1] * pad, positions + [0] * pad, waits), table, free, left


def _plan_case(B, page, hi, add, seed, ended=0.1, spare=None, extra=0):
    g = torch.Generator().manual_seed(seed)
    past = torch.randint(0, hi + 1, (B,), generator=g)
    new = torch.randint(0, add + 1, (B,), generator=g)
    tokens = int(new.sum()) + extra
    new[torch.rand(B, generator=g) < ended] = -1
    width = (hi + add + page - 1) // page
    have = (past + page - 1) // page
    held = int(have.sum())
    need = int(((past + new.clamp(min=0) + page - 1) // page - have).sum())
    spare = need + 3 if spare is None else int(need * spare)
    ids = torch.randperm(held + spare, generator=g)
    table = torch.full((B, width), -1)
    table[torch.arange(width) < have[:, None]] = ids[:held]
    free = torch.cat([ids[held:], torch.full((held,), -1)])
    return past, new, table, free, spare, page, tokens


def _plan_check(case, dev, inplace=True, out=None):
    K = _k()
    past, new, table, free, count, page, tokens = case
    want, wtable, wfree, wleft = _plan_ref(past.tolist(), new.tolist(), table.tolist(), free.tolist(), count, page, tokens)
    i32 = dict(dtype=torch.int32, device=dev)
    wide = torch.full((len(past) + 1, table.shape[1] + 2), 77, **i32)
    t = wide[:len(past), :table.shape[1]]
    t.copy_(table)
    f, c = free.to(**i32), torch.tensor([count], **i32)
    left = c if inplace else torch.empty(1, **i32)
    got = K.paged_plan(past.to(**i32), new.to(**i32), t, f, c, page, tokens, count_out=left, out=out)
    for name, x, w in zip(("lens", "starts", "slots", "rows", "positions", "waits"), got, want):
        assert x.tolist() == w, name
    assert t.tolist() == wtable and f.tolist() == wfree and left.item() == wleft
    assert bool((wide[:, table.shape[1]:] == 77).all()) and bool((wide[-1] == 77).all())
    if not inplace:
        assert c.item() == count
    return got


@pytest.mark.parametrize("B,page,hi,add", [(1, 16, 0, 1), (1, 1, 5, 9), (3, 16, 40, 0), (64, 16, 51, 1), (65, 1, 30, 3),
                                           (200, 8, 100, 40), (1023, 2, 9, 3), (1025, 16, 60, 2), (3000, 16, 20, 5),
                                           (9, 64, 1000, 2000), (2500, 4, 300, 11)])
def test_plan(hip_device, B, page, hi, add):
    _plan_check(_plan_case(B, page, hi, add, 14), hip_device)
    _plan_check(_plan_case(B, page, hi, add, 15, ended=0.6, extra=37), hip_device, inplace=False)


@pytest.mark.parametrize("B,page,hi,add", [(70, 4, 30, 9), (1500, 2, 20, 6), (5, 16, 100, 3000)])
@pytest.mark.parametrize("spare", [0.0, 0.3, 0.9])
def test_plan_without_enough_pages(hip_device, B, page, hi, add, spare):
    got = _plan_check(_plan_case(B, page, hi, add, 16, ended=0.02, spare=spare), hip_device)
    assert got[5].sum() > 0 or spare > 0.5


def test_plan_lengths_that_do_not_fit(hip_device):
    """Negative lengths, lengths past the table, tokens past the step's capacity, every request ended."""
    past, new, table, free, count, page, tokens = _plan_case(40, 8, 50, 9, 17)
    past[3], past[7], new[9], past[11], new[11] = -4, 1 << 30, (1 << 31) - 1, (1 << 31) - 1, (1 << 31) - 1
    past[13], new[13] = -(1 << 31), -5
    _plan_check((past, new, table, free, count, page, tokens), hip_device)
    _plan_check((past, new, table, free, count, page, tokens // 2), hip_device)
    _plan_check((past, new, table, free, count, page, 0), hip_device)
    _plan_check((past, torch.full_like(new, -1), table, free, count, page, 5), hip_device)
    _plan_check((past.clamp(0, 40), new.clamp(0, 9), table, free, -3, page, tokens), hip_device)
    table[:, 0] = 1 << 20  # a page that is not the pool's: no slot
    _plan_check((past, new, table, free, count, page, tokens), hip_device)


def test_plan_outputs_again_and_refusals(hip_device):
    K, dev = _k(), hip_device
    case = _plan_case(30, 16, 50, 3, 18)
    first = _plan_check(case, dev)
    again = _plan_check(case, dev, out=first)
    assert all(a is b for a, b in zip(first, again))
    i32 = dict(dtype=torch.int32, device=dev)
    p, t, c = torch.zeros(2, **i32), torch.zeros(2, 4, **i32), torch.ones(1, **i32)
    ok = dict(past=p, new=p, table=t, free=torch.zeros(8, **i32), count=c, page=16, tokens=4)
    for bad in (dict(past=p.long()), dict(past=p[:1]), dict(table=t.t()), dict(table=t.long()), dict(count=p), dict(page=5),
                dict(tokens=-1), dict(tokens=(1 << 32) + 4), dict(page=(1 << 32) + 16), dict(free=torch.zeros(0, **i32)), dict(count=c.cpu()), dict(out=first),
                dict(new=torch.zeros(4, **i32)[::2])):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            K.paged_plan(**{**ok, **bad})


def test_plan_captured(hip_device):
    """A captured planner (in place: its own count, table and stack go on) against the host's."""
    K, dev = _k(), hip_device
    B, page, width, pool = 12, 4, 16, 100
    i32 = dict(dtype=torch.int32, device=dev)
    past, new, table = torch.zeros(B, **i32), torch.zeros(B, **i32), torch.full((B, width), -1, **i32)
    free, count = torch.randperm(pool).to(**i32), torch.tensor([pool], **i32)
    hpast, htable, hfree, hcount = [0] * B, table.tolist(), free.tolist(), pool
    out = K.paged_plan(past, new, table, free, count, page, 40)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.paged_plan(past, new, table, free, count, page, 40, out=out)
    gen = torch.Generator().manual_seed(19)
    for turn in range(25):
        step = torch.randint(0, 4, (B,), generator=gen)
        step[torch.rand(B, generator=gen) < 0.15] = -1
        new.copy_(step)
        past.copy_(torch.tensor(hpast))
        g.replay()
        want, htable, hfree, hcount = _plan_ref(hpast, step.tolist(), htable, hfree, hcount, page, 40)
        assert [x.tolist() for x in out] == list(want) and table.tolist() == htable
        assert free.tolist() == hfree and count.item() == hcount
        hpast = want[0]


# ---- together -------------------------------------------------------------------------------
@pytest.mark.parametrize("page", [1, 16])
def test_serving_steps(hip_device, page):
    """Requests of different lengths come, grow by a token a step and end; the planner, the writer
    and the attention follow them against dense keys and values kept on the host."""
    K, dev = _k(), hip_device
    B, H, hkv, dh, width, pool = 6, 8, 2, 64, 160 // page, 420 // page
    g = torch.Generator().manual_seed(20)
    i32 = dict(dtype=torch.int32, device=dev)
    table, free = torch.full((B, width), -1, **i32), torch.randperm(pool, generator=g).to(**i32)
    count, lens = torch.tensor([pool], **i32), torch.zeros(B, **i32)
    kc, vc = (torch.full((pool, page, hkv, dh), math.nan, device=dev) for _ in range(2))
    dense = [[] for _ in range(B)]
    for step in range(40):
        new = []
        for b in range(B):
            if not dense[b]:
                new.append(int(torch.randint(0, 60, (1,), generator=g)) if step % 3 == b % 3 else 0)
            else:
                new.append(-1 if len(dense[b]) > 90 else 1)
        total = sum(max(n, 0) for n in new)
        # the pool is smaller than what the requests come to want: some have to wait for others to end
        want = _plan_ref(lens.tolist(), new, table.tolist(), free.tolist(), count.item(), page, total + 2)[0]
        lens, starts, slots, rows, positions, waits = K.paged_plan(lens, torch.tensor(new, **i32), table, free, count,
                                                                   page, total + 2)
        assert waits.tolist() == want[5]
        k, v = (torch.randn(total + 2, hkv, dh, generator=g) for _ in range(2))
        K.paged_write(k.to(dev), v.to(dev), kc, vc, slots)
        for b in range(B):
            if new[b] < 0:
                dense[b] = []
        for i, r in enumerate(rows.tolist()):
            if r >= 0:
                assert positions[i].item() == len(dense[r])
                dense[r].append((k[i], v[i]))
        assert lens.tolist() == [len(d) for d in dense]
        q = torch.randn(B, H, dh, generator=g)
        got = K.paged_attention(q.to(dev), kc, vc, table, lens).cpu().double()
        n = max(len(d) for d in dense)
        if n == 0:
            continue
        dk, dv = (torch.zeros(B, n, hkv, dh) for _ in range(2))
        for b, d in enumerate(dense):
            for j, (x, y) in enumerate(d):
                dk[b, j], dv[b, j] = x, y
        out, _, tol, _ = _reference(q, dk, dv, torch.arange(B).view(B, 1), [len(d) for d in dense], dh ** -0.5)
        assert bool(((got - out).abs() <= tol).all())


def test_plan_in_place_lengths(hip_device):
    """past and the returned lengths are one buffer, step after step, in both launch forms."""
    K, dev = _k(), hip_device
    i32 = dict(dtype=torch.int32, device=dev)
    for B, page, add in ((20, 4, 3), (30, 16, 400), (1500, 8, 2)):
        g = torch.Generator().manual_seed(21)
        width, pool = 4 * (add + page) // page + 2, 0
        pool = B * width
        table, free = torch.full((B, width), -1, **i32), torch.randperm(pool, generator=g).to(**i32)
        count, tokens = torch.tensor([pool], **i32), B * add + 1
        hl, ht, hf, hc = [0] * B, table.tolist(), free.tolist(), pool
        out = None
        lens = torch.zeros(B, **i32)
        for step in range(4):
            new = torch.randint(0, add + 1, (B,), generator=g)
            out = K.paged_plan(lens, new.to(**i32), table, free, count, page, tokens, out=out)
            want, ht, hf, hc = _plan_ref(hl, new.tolist(), ht, hf, hc, page, tokens)
            assert [x.tolist() for x in out] == list(want) and table.tolist() == ht and count.item() == hc
            lens, hl = out[0], want[0]


def test_plan_outputs_at_odd_places(hip_device):
    """Outputs that do not start on 16 bytes, inside wider buffers that stay as they are around them."""
    K, dev = _k(), hip_device
    for case in (_plan_case(9, 64, 1000, 2000, 22), _plan_case(40, 16, 60, 5, 23)):
        past, tokens = case[0], case[6]
        B = len(past)
        bufs = [torch.full((n + 3,), 55, dtype=d, device=dev) for n, d in zip(
            (B, B + 1, tokens, tokens, tokens, B), (torch.int32, torch.int32, torch.int64, torch.int32, torch.int64,
                                                    torch.int32))]
        _plan_check(case, dev, out=tuple(b[1:-2] for b in bufs))
        for b in bufs:
            assert b[0] == 55 and bool((b[-2:] == 55).all())


@pytest.mark.parametrize("B,page,hi,add,width", [(3, 64, 50, 700000, 0), (2, 1, 9, 5, (1 << 20) + 3), (4500, 2, 9, 3, 0),
                                                 (1100, 1, 9, 30, 0)])
def test_plan_large(hip_device, B, page, hi, add, width):
    """More than a million tokens, a table wider than a million pages, more requests than the token pass
    keeps in LDS: the forms with 64-bit sums and a second launch."""
    past, new, table, free, count, page, tokens = _plan_case(B, page, hi, add, 25, ended=0.2, extra=5)
    if width:
        table = torch.cat([table, torch.full((B, width - table.shape[1]), -1)], 1)
    K, i32 = _k(), dict(dtype=torch.int32, device=hip_device)
    short = [r[:max(1, (hi + add) // page + 2)] for r in table.tolist()]
    want, wtable, wfree, wleft = _plan_ref(past.tolist(), new.tolist(), short, free.tolist(), count, page, tokens)
    t, f, c = table.to(**i32), free.to(**i32), torch.tensor([count], **i32)
    got = K.paged_plan(past.to(**i32), new.to(**i32), t, f, c, page, tokens)
    for x, w in zip(got, want):
        assert x.tolist() == w
    n = len(short[0])
    assert t[:, :n].tolist() == [r[:n] for r in wtable] and bool((t[:, n:] == -1).all())
    assert f.tolist() == wfree and c.item() == wleft
