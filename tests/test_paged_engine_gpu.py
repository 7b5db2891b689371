"""The Transformer decoder on the paged cache (decode states beyond 64 positions, or on request) and its
log-probabilities, against the CPU oracle in 64 bits and against the dense cache.

Tolerance of the fp32 model: a logit passes through at most 8 products a layer of at most 128 fp32
terms each, (128 + 2) 2^-24 = 8e-6 relative apiece at worst and random in sign, so 16 of them stay
below 1e-4 of the logits' norm (1.3e-4 if every one were at its worst and of one sign)."""
import functools
import json
import math
import os

import pytest
import torch
from safetensors.torch import load_file

from golden_util import GOLDEN_DIR, make_captions, make_features, make_params, word_map
from oracle import decoders
from test_beam_gpu import _FixedEncoder
from test_greedy_gpu import _decoder as _golden_decoder

pytestmark = pytest.mark.gpu

CFG = dict(d=128, H=2, ff=96, V=101, layers=2, E=72, L=90)


def _rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm()).item()


def _model(dev, dtype=torch.float32, dropout=0.0):
    from imagecaptioningconvnext_amd.models.transformerDecoder import TransformerDecoder
    c = CFG
    dec = TransformerDecoder(embed_dim=c["d"], decoder_dim=c["ff"], vocab_size=c["V"], maxLen=c["L"], device=dev,
                             wordMap=None, pretrained_embeddings_path=None, fine_tune_embeddings=True, dropout=dropout,
                             encoder_dim=c["E"], num_heads=c["H"], num_layers=c["layers"], compute_dtype=dtype)
    p = make_params({n: tuple(q.shape) for n, q in dec.named_parameters()}, 5)
    dec.load_state_dict({**dec.state_dict(), **p})
    return dec.to(dev).eval(), {k: v.double() for k, v in p.items()}


def _oracle(p, enc, caps, lens, pad=None):
    if pad is None:
        pad = torch.zeros_like(caps, dtype=torch.bool)
    return decoders.transformer_tf_forward(p, enc.double(), caps, lens, pad, CFG["H"], CFG["layers"],
                                           pe=decoders.positional_encoding(CFG["d"], CFG["L"]).double())[0]


@pytest.mark.parametrize("pixels", [7, 10])
def test_steps_past_64_positions(hip_device, pixels):
    """Every step's logits over 80 positions (and 49 / 100 pixels) against one pass of the oracle."""
    dec, p = _model(hip_device)
    B, L = 3, 80
    enc = make_features((B, pixels, pixels, CFG["E"]), 6)
    caps = torch.randint(0, CFG["V"], (B, L), generator=torch.Generator().manual_seed(7))
    want = _oracle(p, enc, caps, torch.full((B, 1), L))
    eng = dec.engine()
    st = eng.decode_init(enc.to(hip_device), L)
    assert st["paged"]
    for t in range(L):
        got = eng.decode_step(st, caps[:, t].to(hip_device))[:, :CFG["V"]]
        assert _rel(got, want[:, t]) < 1e-4, t
    with pytest.raises(ValueError, match="full"):
        eng.decode_step(st, caps[:, 0].to(hip_device))


def test_selected_rows_share_pages(hip_device):
    """Rows dropped, reordered, repeated and multiplied on the way: the paged state's logits are the
    dense one's."""
    dec, _ = _model(hip_device)
    eng = dec.engine()
    enc = make_features((4, 7, 7, CFG["E"]), 8).to(hip_device)
    a, b = eng.decode_init(enc, 40), eng.decode_init(enc, 40, paged=True)
    assert not a["paged"] and b["paged"]
    g = torch.Generator().manual_seed(9)
    picks = {3: [3, 1, 1, 0], 7: [2, 2], 11: [0, 1, 0, 1, 1, 0, 0], 20: [6, 5, 4, 3, 2, 1, 0, 0, 1], 30: [8]}
    rows = 4
    for t in range(40):
        if t in picks:
            idx = torch.tensor(picks[t], device=hip_device)
            eng.decode_select(a, idx)
            eng.decode_select(b, idx)
            rows = len(picks[t])
        ids = torch.randint(0, CFG["V"], (rows,), generator=g).to(hip_device)
        x, y = eng.decode_step(a, ids)[:, :CFG["V"]], eng.decode_step(b, ids)[:, :CFG["V"]]
        assert _rel(y, x) < 1e-5, t  # the same sums in fp32 up to their order, two attentions a layer


@pytest.mark.parametrize("k", [3, 5])
def test_beam_search_on_pages(hip_device, k):
    """The reference's beam search result with every decode state on pages."""
    from imagecaptioningconvnext_amd import beam
    t = load_file(os.path.join(GOLDEN_DIR, "beam_small.safetensors"))
    with open(os.path.join(GOLDEN_DIR, "beam_small.json")) as f:
        meta = json.load(f)["trf"]
    cfg = meta["cfg"]
    dec = _golden_decoder(False, cfg, 0.0, hip_device)
    with torch.no_grad():
        dec.fc_out.bias[cfg["V"] - 1] += meta["end_bias_added"]
    eng = dec.engine()
    eng.decode_init = functools.partial(eng.decode_init, paged=True)
    enc = _FixedEncoder(t["trf.feats"].to(hip_device))
    seq, _ = beam.caption_image_beam_search_transformer(enc, dec, torch.zeros(3, 256, 256, dtype=torch.uint8),
                                                        word_map(cfg["V"]), beamSize=k)
    assert seq == t[f"trf.k{k}.seq"].tolist()


def test_greedy_on_pages(hip_device):
    t = load_file(os.path.join(GOLDEN_DIR, "greedy_small.safetensors"))
    with open(os.path.join(GOLDEN_DIR, "greedy_small.json")) as f:
        m = json.load(f)["trf_end"]
    dec = _golden_decoder(False, m["cfg"], m["end_bias_added"], hip_device)
    eng = dec.engine()
    eng.decode_init = functools.partial(eng.decode_init, paged=True)
    preds, seqs = dec(teacherForcing=False, encoder_out=t["trf_end.enc"].to(hip_device), wordMap=word_map(m["cfg"]["V"]),
                      maxDecodeLen=m["maxDecodeLen"])
    assert torch.equal(seqs.cpu(), t["trf_end.sequences"])
    assert _rel(preds, t["trf_end.predictions"]) < 1e-4


def test_bf16_state_agrees_with_the_dense_one(hip_device):
    """bf16: both round a step's activations alike; the attentions' outputs differ in their last bit at
    most (2^-8), which the layers pass on: 2 layers x 2 attentions of it stay below 4 * 2^-8 in norm."""
    dec, _ = _model(hip_device, torch.bfloat16)
    eng = dec.engine()
    enc = make_features((5, 7, 7, CFG["E"]), 10).to(hip_device)
    a, b = eng.decode_init(enc, 20), eng.decode_init(enc, 20, paged=True)
    g = torch.Generator().manual_seed(11)
    for t in range(20):
        ids = torch.randint(0, CFG["V"], (5,), generator=g).to(hip_device)
        assert _rel(eng.decode_step(b, ids)[:, :CFG["V"]], eng.decode_step(a, ids)[:, :CFG["V"]]) < 4 * 2.0 ** -8


def test_refusals(hip_device):
    dec, _ = _model(hip_device, dropout=0.1)
    eng = dec.engine()
    enc = make_features((2, 7, 7, CFG["E"]), 12).to(hip_device)
    with pytest.raises(ValueError, match="64"):
        eng.decode_init(enc, 65, paged=False)
    with pytest.raises(ValueError, match="positional"):
        eng.decode_init(enc, CFG["L"] + 1)
    st = eng.decode_init(enc, 70)
    ids = torch.zeros(2, dtype=torch.int64, device=hip_device)
    eng.cross_probs = []
    with pytest.raises(ValueError, match="probabilities"):
        eng.decode_step(st, ids)
    eng.cross_probs = None
    dec.train()
    with pytest.raises(ValueError, match="eval"):
        eng.decode_init(enc, 70)
    with pytest.raises(ValueError, match="probabilities"):
        eng.decode_step(st, ids)


@pytest.mark.parametrize("masked", [False, True])
def test_log_probs_and_gradients(hip_device, masked):
    """logProbs and the gradients of every parameter and the encoder's output, against autograd through
    the oracle in 64 bits."""
    dec, p = _model(hip_device)
    B, L, V = 4, 14, CFG["V"]
    caps, lens = make_captions(B, L, [14, 9, 3, 12], V, 13)
    enc = make_features((B, 7, 7, CFG["E"]), 14)
    pad = (caps == 0) if masked else torch.zeros_like(caps, dtype=torch.bool)
    gen = torch.Generator().manual_seed(15)
    g, h = torch.randn(B, L, generator=gen), torch.randn(B, L, generator=gen)
    live = torch.arange(L) < lens - 1
    x = enc.to(hip_device).requires_grad_(True)
    logp, ent, tl, ti = dec.logProbs(x, caps.to(hip_device), lens.to(hip_device), pad.to(hip_device) if masked else None, top=4)
    (logp * g.to(hip_device) + ent * (h * live).to(hip_device)).sum().backward()
    pr = {k: v.clone().requires_grad_(True) for k, v in p.items()}
    ex = enc.double().requires_grad_(True)
    logq = torch.log_softmax(_oracle(pr, ex, caps, lens, pad), -1)
    nxt = torch.where(live, torch.roll(caps, -1, 1), 0)
    wlogp = torch.where(live, logq.gather(-1, nxt[..., None])[..., 0], 0.0)
    went = -(logq.exp() * logq).sum(-1)
    (wlogp * g + went * h * live).sum().backward()
    assert _rel(logp, wlogp) < 1e-4 and _rel(ent, went) < 1e-4
    assert bool((logp.detach().cpu()[~live] == 0).all())
    best = logq.detach().topk(4, -1)
    near = (best.values[..., :-1] - best.values[..., 1:]).amin() > 1e-4  # no alternatives closer than the logits' error
    assert not near or torch.equal(ti.cpu(), best.indices)
    assert _rel(tl, best.values) < 1e-4
    assert _rel(x.grad, ex.grad) < 1e-4
    params = dict(dec.named_parameters())
    for name, q in pr.items():
        assert _rel(params[name].grad, q.grad) < 1e-4, name


@pytest.mark.parametrize("loss", ["mean", "weighted"])
@pytest.mark.parametrize("masked", [False, True])
def test_entropy_gradient_is_that_of_every_position(hip_device, masked, loss):
    """The entropy of the positions past a caption's last target has a value, so it has a gradient too: a
    loss over all positions (a mean, whose gradient comes expanded, and one of its own weights) against
    autograd through the oracle in 64 bits.  logp there is 0 whatever the parameters are."""
    dec, p = _model(hip_device)
    B, L = 4, 14
    caps, lens = make_captions(B, L, [14, 9, 3, 12], CFG["V"], 13)
    enc = make_features((B, 7, 7, CFG["E"]), 14)
    pad = (caps == 0) if masked else torch.zeros_like(caps, dtype=torch.bool)
    h = torch.randn(B, L, generator=torch.Generator().manual_seed(18))
    live = torch.arange(L) < lens - 1

    def value(logp, ent, w):
        return logp.sum() / 20 + ent.mean() if loss == "mean" else (logp * w + ent * w).sum()

    x = enc.to(hip_device).requires_grad_(True)
    logp, ent, _, _ = dec.logProbs(x, caps.to(hip_device), lens.to(hip_device), pad.to(hip_device) if masked else None)
    value(logp, ent, h.to(hip_device)).backward()
    pr = {k: v.clone().requires_grad_(True) for k, v in p.items()}
    ex = enc.double().requires_grad_(True)
    logq = torch.log_softmax(_oracle(pr, ex, caps, lens, pad), -1)
    wlogp = torch.where(live, logq.gather(-1, torch.where(live, torch.roll(caps, -1, 1), 0)[..., None])[..., 0], 0.0)
    value(wlogp, -(logq.exp() * logq).sum(-1), h.double()).backward()
    assert _rel(x.grad, ex.grad) < 1e-4
    params = dict(dec.named_parameters())
    for name, q in pr.items():
        assert _rel(params[name].grad, q.grad) < 1e-4, name


def test_outputs_changed_by_the_caller_leave_the_backward_alone(hip_device):
    """The tensors that logprobs returns are the caller's: the backward does not read them again."""
    dec, _ = _model(hip_device)
    B, L = 3, 12
    caps, lens = make_captions(B, L, [12, 5, 8], CFG["V"], 19)
    enc = make_features((B, 7, 7, CFG["E"]), 20).to(hip_device)
    eng = dec.engine()
    gen = torch.Generator().manual_seed(21)
    g, h = (torch.randn(B, L, generator=gen).to(hip_device) for _ in range(2))
    grads = []
    for change in (False, True):
        s = eng.forward(enc, caps.to(hip_device), lens.to(hip_device), loss=False)
        out = eng.logprobs(s, 3)
        if change:
            for t in out:
                t.fill_(7)
        buf = torch.empty_like(eng.fp.grad)
        eng.logprobs_backward(s, g, h, gbuf=buf)
        grads.append(buf)
    assert torch.equal(*grads)


def test_log_probs_changed_in_place(hip_device):
    """Padding masked out in place, as logits and losses usually are: the same gradients as out of place,
    and a second backward through the same graph gives them again."""
    dec, _ = _model(hip_device)
    B, L = 3, 12
    caps, lens = make_captions(B, L, [12, 5, 8], CFG["V"], 19)
    enc = make_features((B, 7, 7, CFG["E"]), 20).to(hip_device)
    dead = (torch.arange(L) >= lens - 1).to(hip_device)
    params = list(dec.parameters())

    def grads(inplace, times=1):
        logp, ent, tl, ti = dec.logProbs(enc, caps.to(hip_device), lens.to(hip_device), top=2)
        assert logp.shape == ent.shape == (B, L) and tl.shape == ti.shape == (B, L, 2) and not tl.requires_grad
        if inplace:
            ent[dead] = 0
            logp.mul_(2)
            tl[dead] = -1
        else:
            ent, logp = torch.where(dead, 0.0, ent), 2 * logp
        for i in range(times):
            g = torch.autograd.grad(logp.sum() + ent.sum(), params, retain_graph=i + 1 < times)
        return g

    want = grads(False)
    for got in (grads(True), grads(True, 2)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_log_probs_are_those_of_the_predictions(hip_device):
    """bf16 at the captions' own width: the fused pass against log_softmax of the same bf16 logits."""
    dec, _ = _model(hip_device, torch.bfloat16)
    B, L = 3, 20
    caps, lens = make_captions(B, L, [20, 5, 11], CFG["V"], 16)
    enc = make_features((B, 7, 7, CFG["E"]), 17).to(hip_device)
    eng = dec.engine()
    with torch.no_grad():
        s = eng.forward(enc, caps.to(hip_device), lens.to(hip_device), loss=False)
        logp, ent, tl, ti = eng.logprobs(s, 5)
    logits = s["logprobs"][0][:, :CFG["V"]].double().cpu().view(B, L, -1)
    logq = torch.log_softmax(logits, -1)
    live = torch.arange(L) < lens - 1
    want = torch.where(live, logq.gather(-1, torch.where(live, torch.roll(caps, -1, 1), 0)[..., None])[..., 0], 0.0)
    assert (logp.cpu().double() - want).abs().max() < 2e-6  # fp32 of values below 16: 4 half steps of 2^-21
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[..., :5]
    assert torch.equal(ti.cpu(), order)


def test_alternatives_are_the_best_words(hip_device):
    """Every position's alternatives against the oracle's order: the same word wherever no other is within
    the logits' error (1e-4 of a row's norm, at the top of this file), which most positions are, and one
    of the same value within it everywhere."""
    dec, p = _model(hip_device)
    B, L, V, top = 4, 14, CFG["V"], 4
    caps, lens = make_captions(B, L, [14, 9, 3, 12], V, 13)
    enc = make_features((B, 7, 7, CFG["E"]), 14)
    with torch.no_grad():
        _, _, tl, ti = dec.logProbs(enc.to(hip_device), caps.to(hip_device), lens.to(hip_device), top=top)
    logits = _oracle(p, enc, caps, lens)
    best = logits.topk(top + 1, -1)
    room = 1e-4 * logits.norm(dim=-1, keepdim=True)
    ti = ti.cpu()
    assert bool(((logits.gather(-1, ti) - best.values[..., :top]).abs() <= room).all())
    assert all(len(set(r)) == top for r in ti.view(-1, top).tolist())
    gaps = best.values[..., :-1] - best.values[..., 1:]
    alone = (gaps > room) & torch.cat([torch.ones(B, L, 1, dtype=torch.bool), (gaps > room)[..., :-1]], -1)
    assert alone.double().mean() > 0.75
    assert torch.equal(ti[alone], best.indices[..., :top][alone])


def _ending(eng, end, offset):
    """Steps whose end word's logit is moved by offset(position)."""
    step = eng.decode_step

    def moved(st, ids):
        t, logits = st["t"], step(st, ids)
        logits[:, end] += offset(t)
        return logits

    eng.decode_step = moved


def _plain_beam(p, enc, start, end, k, most, offset):
    """Beam search that decodes every prefix again with the oracle: (words, the steps at which beams ended,
    the least distance of a kept score to the next one)."""
    rows, scores, done, ends, gap = [[start]], torch.zeros(1, dtype=torch.float64), [], [], math.inf
    for t in range(most):
        caps = torch.tensor(rows)
        logits = _oracle(p, enc.expand(len(rows), -1, -1, -1), caps, torch.full((len(rows), 1), t + 2))[:, -1].clone()
        logits[:, end] += offset(t)
        best = torch.sort((scores[:, None] + torch.log_softmax(logits, -1)).view(-1), descending=True, stable=True)
        gap = min(gap, (best.values[:k] - best.values[1:k + 1]).min().item())
        new = [(rows[i // CFG["V"]] + [i % CFG["V"]], v) for i, v in zip(best.indices[:k].tolist(), best.values)]
        done += [r for r in new if r[0][-1] == end]
        ends += [t for r in new if r[0][-1] == end]
        new = [r for r in new if r[0][-1] != end]
        k = len(new)
        if not k:
            break
        rows, scores = [r[0] for r in new], torch.stack([r[1] for r in new])
    return max(done, key=lambda r: r[1])[0], ends, gap


@pytest.mark.parametrize("k,seed,ends", [(3, 22, [72, 73, 73]), (4, 36, [71, 72, 72, 72])])
def test_beam_search_past_64_positions(hip_device, k, seed, ends):
    """Captions of more than 70 words: no beam may end before position 66, then they end one after another.
    Scores closer than 5e-4, some thousand times their error in fp32, would not be a test of the search."""
    from imagecaptioningconvnext_amd import beam
    dec, p = _model(hip_device)
    V, enc = CFG["V"], make_features((1, 7, 7, CFG["E"]), seed)

    def offset(t):
        return -1e4 if t < 66 else 0.02 * (t - 66) - 0.1

    with torch.no_grad():
        want, at, gap = _plain_beam(p, enc, V - 2, V - 1, k, 88, offset)
    assert at == ends and gap > 5e-4
    _ending(dec.engine(), V - 1, offset)
    seq, _ = beam.caption_image_beam_search_transformer(_FixedEncoder(enc.to(hip_device)), dec,
                                                        torch.zeros(3, 256, 256, dtype=torch.uint8), word_map(V),
                                                        beamSize=k, max_decode_len=88)
    assert seq == want


def test_greedy_past_64_positions(hip_device):
    """No row ends before position 66; from 70 on every row does.  Logits of every step against one pass of
    the oracle over the words chosen, which are its best ones."""
    dec, p = _model(hip_device)
    B, L, V = 3, 80, CFG["V"]
    enc = make_features((B, 7, 7, CFG["E"]), 37)

    def offset(t):
        return -1e4 if t < 66 else 0.0 if t < 70 else 1e4

    _ending(dec.engine(), V - 1, offset)
    preds, seqs = dec(teacherForcing=False, encoder_out=enc.to(hip_device), wordMap=word_map(V), maxDecodeLen=L)
    preds, seqs = preds.cpu().double(), seqs.cpu()
    caps = torch.cat([torch.full((B, 1), V - 2), seqs[:, :-1]], 1)
    want = _oracle(p, enc, caps, torch.full((B, 1), L))
    for b in range(B):
        n = seqs[b].tolist().index(V - 1) + 1  # words with the end
        assert 67 <= n <= 71
        moved = want[b, :n] + torch.tensor([[offset(t) * (w == V - 1) for w in range(V)] for t in range(n)], dtype=torch.float64)
        words = torch.arange(V) != V - 1
        assert _rel(preds[b, :n][:, words], moved[:, words]) < 1e-4
        room = 1e-4 * want[b, :n].norm(dim=-1)
        assert bool((moved.gather(-1, seqs[b, :n, None])[:, 0] >= moved.amax(-1) - room).all())
        assert bool((preds[b, n:] == 0).all())
