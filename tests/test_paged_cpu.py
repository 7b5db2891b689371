"""Refusals of the paged-cache and token log-probability entry points at the C boundary: every call
here is turned down before anything is launched (there is no GPU), with a message that says why."""
import ctypes

import pytest
import torch

from imagecaptioningconvnext_amd import _abi
from imagecaptioningconvnext_amd import kernels as K

A = 1 << 20  # an aligned address that is never read: the calls are refused on the host


def _attn(**kw):
    d = _abi.PagedAttnDesc(_abi.BF16, 2, 8, 2, 64, 16, 10, 4, 64, 0.125, 512, 64, 512, 64, 2048, 128, 64, 2048, 128, 64,
                           4, A, A, A, A, None, A, A, None, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _said():
    return _abi.lib().imgcap_last_error_string().decode()


@pytest.mark.parametrize("kw,why", [
    (dict(dtype=2), "dtype"), (dict(dh=96), "head dim"), (dict(dh=0), "head dim"), (dict(H=9), "multiple"),
    (dict(Hkv=0), "multiple"), (dict(H=0), "multiple"), (dict(B=-1), "multiple"), (dict(page=12), "power of two"),
    (dict(page=0), "power of two"), (dict(page=2048), "power of two"), (dict(pages=0), "empty"), (dict(width=0), "empty"),
    (dict(max_len=0), "empty"), (dict(max_len=65), "max_len"), (dict(width=1 << 30), "2^31"), (dict(q=None), "NULL"),
    (dict(k=None), "NULL"), (dict(lens=None), "NULL"), (dict(table=None), "NULL"), (dict(o=None), "NULL"),
    (dict(q=A + 2), "16-byte"), (dict(v=A + 8), "16-byte"), (dict(k_tok=129), "16"), (dict(v_head=60), "16"),
    (dict(q_row=511), "16"), (dict(k_page=2047), "16"),
])
def test_attention_refuses(kw, why):
    d, need = _attn(**kw), ctypes.c_int64(-1)
    assert _abi.lib().imgcap_paged_attention(ctypes.byref(d), None) == -1
    assert why in _said()
    assert _abi.lib().imgcap_paged_attention_ws(ctypes.byref(d), ctypes.byref(need)) == -1
    assert need.value == -1


def test_attention_needs_its_workspace():
    """A split length without the workspace is refused as such, and the size asked for is enough to
    hold a maximum, a sum and an output per part."""
    d, need = _attn(width=4096, max_len=65536), ctypes.c_int64(0)
    assert _abi.lib().imgcap_paged_attention_ws(ctypes.byref(d), ctypes.byref(need)) == 0
    assert need.value >= 2 * 8 * 2 * (64 + 2) * 4
    for ws, size in ((None, need.value), (A + 4, need.value), (A, need.value - 1)):
        d.ws, d.ws_bytes = ws, size
        assert _abi.lib().imgcap_paged_attention(ctypes.byref(d), None) == _abi.IMGCAP_EWORKSPACE
    assert _abi.lib().imgcap_paged_attention(None, None) == -1
    empty = _attn(B=0)
    assert _abi.lib().imgcap_paged_attention(ctypes.byref(empty), None) == 0


MOST = (1 << 31) - 65536  # positions of the widest table


@pytest.mark.parametrize("max_len", [MOST, MOST - 1, MOST - 31, 2130706432, 1900000000, 1200000000, 1 << 30, 600000, 4097])
@pytest.mark.parametrize("B", [1, 2, 17, 128, 1000, 2047])
def test_attention_workspace_of_long_lengths(B, max_len):
    """Lengths near the bound, whose sum with a part's length passes 32 bits: the workspace is a maximum, a
    sum and an output per part, of 2 to 1024 parts, where the rows alone are fewer than half of the
    4096 workgroups that the length is cut for."""
    d, need = _attn(B=B, H=1, Hkv=1, page=1024, width=(MOST + 1023) // 1024, max_len=max_len), ctypes.c_int64(0)
    assert _abi.lib().imgcap_paged_attention_ws(ctypes.byref(d), ctypes.byref(need)) == 0
    parts, rest = divmod(need.value, B * (64 + 2) * 4)
    assert rest == 0 and 2 <= parts <= 1024
    assert _abi.lib().imgcap_paged_attention(ctypes.byref(d), None) == _abi.IMGCAP_EWORKSPACE


@pytest.mark.parametrize("kw", [
    dict(B=1 << 24, H=1, Hkv=1, max_len=33, dtype=_abi.F32), dict(B=1 << 24, H=1, Hkv=1, width=5, max_len=65),
    dict(B=1 << 21, H=8, Hkv=8, width=64, max_len=1000), dict(B=1 << 22, H=34, Hkv=2, width=5, max_len=65),
    dict(B=1 << 26, H=1, Hkv=1), dict(B=1 << 30, H=1 << 30, Hkv=1 << 30), dict(B=(1 << 31) - 1, H=(1 << 31) - 1, Hkv=1),
])
def test_attention_refuses_more_rows_than_a_launch_takes(kw):
    """A launch has fewer than 2^32 threads; row counts whose products pass 63 bits with the length."""
    d, need = _attn(**kw), ctypes.c_int64(-1)
    assert _abi.lib().imgcap_paged_attention(ctypes.byref(d), None) == -1
    assert "too many rows" in _said()
    assert _abi.lib().imgcap_paged_attention_ws(ctypes.byref(d), ctypes.byref(need)) == -1
    assert need.value == -1


@pytest.mark.parametrize("kw", [
    dict(n=1 << 24), dict(n=(1 << 31) - 1), dict(n=1 << 23, V=40000, ld=40000), dict(n=1 << 24, V=32761, ld=32761),
    dict(n=1 << 23, V=16390, ld=16390, dtype=_abi.F32),
])
def test_logprobs_refuse_more_rows_than_a_launch_takes(kw):
    assert _abi.lib().imgcap_token_logprobs(ctypes.byref(_logprobs(**kw)), None) == -1
    assert "too many rows" in _said()


@pytest.mark.parametrize("kw", [
    dict(n=1 << 24), dict(n=1 << 23, V=9490, ldd=9490, ld=9490), dict(n=1 << 20, V=131072, ld=131072, ldd=131072),
    dict(n=1 << 23, V=5000, ld=5000, ldd=5000, dtype=_abi.F32),
])
def test_logprobs_bwd_refuses_more_rows_than_a_launch_takes(kw):
    assert _abi.lib().imgcap_token_logprobs_bwd(ctypes.byref(_logprobs(**kw)), None) == -1
    assert "too many rows" in _said()


@pytest.mark.parametrize("kw,why", [
    (dict(dtype=3), "dtype"), (dict(dh=60), "16-byte"), (dict(heads=0), "16-byte"), (dict(n=-1), "16-byte"),
    (dict(page=24), "power of two"), (dict(pages=0), "power of two"), (dict(k=None), "NULL"), (dict(slots=None), "NULL"),
    (dict(k_row=4), "strides"), (dict(vc_tok=12), "strides"), (dict(vc=A + 4), "aligned"), (dict(n=1 << 30), "2^31"),
])
def test_write_refuses(kw, why):
    d = _abi.PagedWriteDesc(_abi.BF16, 3, 8, 64, 16, 10, 512, 64, 512, 64, 8192, 512, 64, 8192, 512, 64, A, A, A, A, A)
    for k, v in kw.items():
        setattr(d, k, v)
    assert _abi.lib().imgcap_paged_write(ctypes.byref(d), None) == -1
    assert why in _said()


def test_write_of_nothing_is_nothing():
    d = _abi.PagedWriteDesc(_abi.F32, 0, 8, 64, 16, 10, *([0] * 10), None, None, None, None, None)
    assert _abi.lib().imgcap_paged_write(ctypes.byref(d), None) == 0


@pytest.mark.parametrize("kw,why", [
    (dict(B=0), "positive"), (dict(width=0), "positive"), (dict(pool=0), "positive"), (dict(tokens=-1), "positive"),
    (dict(page=3), "power of two"), (dict(page=4096), "power of two"), (dict(width=1 << 28, table_row=1 << 28), "2^31"),
    (dict(table_row=3), "overlap"), (dict(past=None), "NULL"), (dict(slots=None), "NULL"),
    (dict(ws=None, tokens=4097), "NULL"), (dict(ws=None, B=1025), "NULL"),
    (dict(ws=None, width=(1 << 20) + 1, table_row=(1 << 20) + 1), "NULL"),
])
def test_plan_refuses(kw, why):
    d = _abi.PagedPlanDesc(2, 4, 16, 8, 2, 4, *([A] * 13))
    for k, v in kw.items():
        setattr(d, k, v)
    assert _abi.lib().imgcap_paged_plan(ctypes.byref(d), None) == -1
    assert why in _said()
    assert _abi.lib().imgcap_paged_plan(None, None) == -1


def _logprobs(**kw):
    d = _abi.LogprobDesc(_abi.BF16, 4, 100, 3, 100, 100, *([A] * 10))
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,why", [
    (dict(dtype=2), "dtype"), (dict(top=65), "top"), (dict(V=8, top=9), "top"), (dict(top=-1), "top"), (dict(V=0), "bad"),
    (dict(n=-1), "bad"), (dict(ld=99), "bad"), (dict(top_logp=None), "NULL"), (dict(top_ids=None), "NULL"),
    (dict(logp=None), "NULL"), (dict(stats=None), "NULL"), (dict(logits=None), "NULL"), (dict(entropy=None), "NULL"),
])
def test_logprobs_refuses(kw, why):
    assert _abi.lib().imgcap_token_logprobs(ctypes.byref(_logprobs(**kw)), None) == -1
    assert why in _said()
    assert _abi.lib().imgcap_token_logprobs(None, None) == -1


@pytest.mark.parametrize("kw,why", [
    (dict(dtype=2), "dtype"), (dict(ldd=99), "bad"), (dict(ld=99), "bad"), (dict(targets=None), "NULL"),
    (dict(stats=None), "NULL"), (dict(entropy=None), "NULL"), (dict(dlogits=None), "NULL"), (dict(ldd=104), "in place"),
])
def test_logprobs_bwd_refuses(kw, why):
    assert _abi.lib().imgcap_token_logprobs_bwd(ctypes.byref(_logprobs(**kw)), None) == -1
    assert why in _said()
    assert _abi.lib().imgcap_token_logprobs_bwd(None, None) == -1


def test_no_rows_is_nothing():
    d = _abi.LogprobDesc(_abi.F32, 0, 10, 3, 10, 10)
    assert _abi.lib().imgcap_token_logprobs(ctypes.byref(d), None) == 0
    assert _abi.lib().imgcap_token_logprobs_bwd(ctypes.byref(d), None) == 0


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 8, 64)
    c = torch.zeros(4, 16, 8, 64)
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 4, dtype=torch.int32)
    for call in (lambda: K.paged_attention(x, c, c, t, i), lambda: K.paged_write(x, x, c, c, i.long()),
                 lambda: K.paged_plan(i, i, t, i, i[:1], 16, 2), lambda: K.token_logprobs(x[0]),
                 lambda: K.token_logprobs_bwd(x[0], None, x[0], x[0, 0])):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


FAR = (1 << 32) + 1  # one, in 32 bits


def _calls_past_32_bits():
    def rows(n, *shape, dtype=torch.float32):  # n of them, all the same
        return torch.zeros(1, *shape, dtype=dtype).expand(n, *(-1 for _ in shape))

    i32 = dict(dtype=torch.int32)
    q, c, t, i = torch.zeros(1, 1, 64), torch.zeros(2, 16, 1, 64), torch.zeros(1, 4, **i32), torch.zeros(1, **i32)

    def meta(*shape, dtype=torch.int32):  # no memory behind it
        return torch.empty(*shape, dtype=dtype, device="meta")

    return {
        "attention, pages": lambda: K.paged_attention(q, rows(FAR, 16, 1, 64), rows(FAR, 16, 1, 64), t, i, out=q),
        "attention, heads": lambda: K.paged_attention(rows(FAR, 64)[None], c, c, t, i, out=rows(FAR, 64)[None]),
        "attention, width": lambda: K.paged_attention(q, c, c, meta(1, FAR), i, max_len=5, out=q),
        "write, pages": lambda: K.paged_write(q, q, rows(FAR, 16, 1, 64), rows(FAR, 16, 1, 64), i.long()),
        "write, heads": lambda: K.paged_write(*[rows(FAR, 64)[None]] * 2, *[c.expand(2, 16, FAR, 64)] * 2, i.long()),
        "plan, pool": lambda: K.paged_plan(i, i, t, meta(FAR), i, 16, 2),
        "plan, rows": lambda: K.paged_plan(meta(FAR), meta(FAR), meta(FAR, 4), i, i, 16, 2),
        "plan, width": lambda: K.paged_plan(i, i, meta(1, FAR), i, i, 16, 2),
        "logprobs, rows": lambda: K.token_logprobs(rows(FAR, 4)),
        "logprobs, words": lambda: K.token_logprobs(meta(1, FAR, dtype=torch.float32)),
    }


@pytest.mark.parametrize("what", list(_calls_past_32_bits()))
def test_wrappers_refuse_counts_past_32_bits(monkeypatch, what):
    """Counts whose low 32 bits are an ordinary number never reach the descriptors, which would keep those."""
    went = []
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda t, *a, **k: torch.empty(0))
    monkeypatch.setattr(K, "_run_on", lambda *a: went.append(a) or 0)
    with pytest.raises(ValueError, match="out of range"):
        _calls_past_32_bits()[what]()
    assert not went


def _attention_calls(monkeypatch, B, H, max_len):
    """The descriptors that a paged_attention of CPU tensors would launch, and the error text before and after."""
    seen = []

    def run(dev, name, d):
        seen.append((name, d.max_len, d.ws_bytes, bool(d.ws)))
        return 0

    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(K, "_run_on", run)
    width = (max_len + 15) // 16
    q, c = torch.zeros(B, H, 64), torch.zeros(1, 16, 1, 64)
    t, i = torch.zeros(1, width, dtype=torch.int32).expand(B, width), torch.zeros(B, dtype=torch.int32)
    K.paged_attention(q, c, c, t, i, max_len=max_len)
    return seen


@pytest.mark.parametrize("B,H,max_len", [(1, 1, 513), (2, 16, 5000), (1, 3, 100000), (300, 1, 1024), (300, 1, 1025), (1, 1, 512)])
def test_attention_is_called_once_with_its_workspace(monkeypatch, B, H, max_len):
    """A split length is no call that fails first: one launch, with the bytes that the size query says."""
    d, need = _attn(dtype=_abi.F32, B=B, H=H, Hkv=1, width=(max_len + 15) // 16, max_len=max_len), ctypes.c_int64(0)
    assert _abi.lib().imgcap_paged_attention_ws(ctypes.byref(d), ctypes.byref(need)) == 0
    _abi.lib().imgcap_paged_attention_ws(None, ctypes.byref(need))  # leaves an error text
    before = _said()
    assert _attention_calls(monkeypatch, B, H, max_len) == [("imgcap_paged_attention", max_len, need.value, need.value > 0)]
    assert _said() == before


@pytest.mark.parametrize("dtype", [_abi.BF16, _abi.F32])
@pytest.mark.parametrize("B", [1, 7, 255, 256, 4096, 1 << 20])
def test_short_lengths_take_no_workspace(dtype, B):
    """What the wrapper takes for granted (_ATTN_WHOLE)."""
    need = ctypes.c_int64(-1)
    for max_len in (1, 32, 33, 64, 65, 500, K._ATTN_WHOLE):
        d = _attn(dtype=dtype, B=B, width=64, max_len=max_len)
        assert _abi.lib().imgcap_paged_attention_ws(ctypes.byref(d), ctypes.byref(need)) == 0
        assert need.value == 0
