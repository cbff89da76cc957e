"""Refusals of the block-scaled 8-bit operators and of the balance loss: every malformed request
is turned down with DMOE_ERR_INVALID and a message before anything reaches a GPU."""

import ctypes
import subprocess
import sys

import pytest
import torch

from distributedmoe_b200 import _native as N

P = ctypes.c_void_p(4096)  # an aligned non-null pointer that a refused call never follows
ODD = ctypes.c_void_p(4100)
NINE = ctypes.c_void_p(4099)


def _refused(rc, words):
    assert rc == 1
    assert words in N.lib().dmoe_last_error().decode(), N.lib().dmoe_last_error()


def _quantize(x=P, dtype=2, batch=1, rows=4, cols=256, block=1, q=P, q_ld=256, s=P, s_ld=2):
    return N.lib().dmoe_quantize_blocks_e4m3(x, dtype, batch, rows, cols, block, q, q_ld, s, s_ld, None)


@pytest.mark.parametrize("kw,words", [
    (dict(dtype=3), "dtype"), (dict(block=64), "block_rows"), (dict(cols=24), "multiple of 16"), (dict(cols=0), "multiple"), (dict(cols=1 << 27, q_ld=1 << 27, s_ld=1 << 20), "2^26"),
    (dict(rows=-1), "multiple of 16"), (dict(x=None), "null"), (dict(q=None), "null"), (dict(s=None), "null"),
    (dict(x=ODD), "aligned"), (dict(q=ODD), "aligned"), (dict(s=NINE), "aligned"), (dict(q_ld=240), "q_ld"),
    (dict(q_ld=264), "q_ld"), (dict(s_ld=1), "scale_ld"), (dict(block=128, q_ld=272), "packed"),
    (dict(block=128, s_ld=3), "packed"), (dict(batch=1 << 40, rows=1 << 40), "rows"),
    (dict(rows=1 << 40), "rows"), (dict(block=128, rows=1 << 40), "blocks"),
])
def test_quantize_refuses(kw, words):
    _refused(_quantize(**kw), words)


def _i32(*v):
    return (ctypes.c_int32 * max(1, len(v)))(*v)


def _matmul(x=P, x_ld=256, xs=P, xs_ld=2, w=P, ws=P, E=2, Nn=64, K=256, experts=(0, 1), ends=(3, 8), n=None, dev=0, m=8,
            hint=0, y=P, y_ld=64, dt=2, status=P):
    a, b = _i32(*experts), _i32(*ends)
    return N.lib().dmoe_grouped_matmul_fp8_blocks(
        x, x_ld, xs, xs_ld, w, ws, E, Nn, K, ctypes.addressof(a), ctypes.addressof(b), len(ends) if n is None else n,
        dev, m, hint, y, y_ld, dt, status, None)


@pytest.mark.parametrize("kw,words", [
    (dict(dt=3), "dtype"), (dict(Nn=60), "multiple of 8"), (dict(K=200), "of 16"), (dict(K=0), "of 16"),
    (dict(E=0), "E_stack"), (dict(m=-1), "m_rows"), (dict(n=-1), "n_seg"), (dict(hint=-1), "rows_hint"),
    (dict(x_ld=240), "x_ld"), (dict(x_ld=264), "x_ld"), (dict(xs_ld=1), "xs_ld"), (dict(y_ld=56), "y_ld"),
    (dict(y_ld=68), "y_ld"), (dict(x=None), "null"), (dict(xs=None), "null"), (dict(w=None), "null"),
    (dict(ws=None), "null"), (dict(y=None), "null"), (dict(status=None), "null"), (dict(x=ODD), "aligned"),
    (dict(w=ODD), "aligned"), (dict(y=ODD), "aligned"), (dict(ws=NINE), "aligned"), (dict(ends=(5, 3)), "segment 1 end"),
    (dict(ends=(3, 9)), "segment 1 end"), (dict(experts=(0, 2)), "expert 2"), (dict(experts=(-1, 0)), "expert -1"),
    (dict(n=257), "257"), (dict(n=1025, dev=1), "1025"), (dict(m=2**31 - 1), "rows or tiles"), (dict(m=2**30, Nn=1 << 20, y_ld=1 << 20), "tiles"),
])
def test_matmul_refuses(kw, words):
    _refused(_matmul(**kw), words)


def _mlp(x=P, x_ld=256, xs=P, xs_ld=2, w=P, ws=P, wd=P, E=2, d=256, inner=128, experts=(0, 1), ends=(3, 8), m=8, hint=0,
         act=1, y=P, work=P, work_bytes=1 << 20, status=P):
    a, b = _i32(*experts), _i32(*ends)
    return N.lib().dmoe_grouped_gated_mlp_fp8_blocks(
        x, x_ld, xs, xs_ld, w, ws, w, ws, wd, ws, E, d, inner, ctypes.addressof(a), ctypes.addressof(b), len(ends), 0, m,
        hint, act, y, work, work_bytes, status, None)


@pytest.mark.parametrize("kw,words", [
    (dict(act=2), "activation"), (dict(d=200, x_ld=256), "multiples of 16"), (dict(inner=24), "multiples of 16"),
    (dict(x_ld=240), "x_ld"), (dict(xs_ld=1), "xs_ld"), (dict(x=None), "null"), (dict(xs=None), "null"),
    (dict(w=None), "null"), (dict(wd=None), "null"), (dict(y=None), "null"), (dict(work=None), "null"),
    (dict(status=None), "null"), (dict(work_bytes=100), "workspace"), (dict(work=ODD), "aligned"), (dict(y=ODD), "aligned"),
    (dict(xs=NINE), "aligned"), (dict(ends=(9, 9)), "segment 0 end"), (dict(experts=(0, 5)), "expert 5"),
])
def test_mlp_refuses(kw, words):
    _refused(_mlp(**kw), words)


def test_empty_requests_are_fine():
    assert _quantize(rows=0) == 0 and _quantize(batch=0) == 0
    assert _matmul(m=0, ends=(0, 0)) == 0 and _matmul(n=0) == 0
    assert _mlp(m=0, ends=(0, 0)) == 0
    assert N.lib().dmoe_balance_loss_backward(None, 0, 0, 8, 2, 0, None, 1, None, P, None, None, None, None) == 0


def _balance(logits=P, dt=0, idx=P, T=16, E=8, k=2, mode=0, seq=None, n=1, mask=None, counts=P, out=None, loss=P, ws=P,
             ws_bytes=1 << 20, status=P):
    return N.lib().dmoe_balance_loss(logits, dt, idx, T, E, k, mode, seq, n, mask, counts, out, loss, ws, ws_bytes, status,
                                     None)


@pytest.mark.parametrize("kw,words", [
    (dict(dt=3), "logits must be"), (dict(mode=2), "mode"), (dict(E=0), "E=0"), (dict(E=1025), "E=1025"),
    (dict(k=0), "k=0"), (dict(k=9), "k=9"), (dict(T=-1), "T=-1"), (dict(n=2), "n_seq=2"), (dict(n=-1, seq=P), "n_seq"),
    (dict(n=(1 << 20) + 1, seq=P), "n_seq"), (dict(T=1 << 30), "too many"),
    (dict(logits=None), "null"), (dict(idx=None), "null"), (dict(counts=None), "null"), (dict(loss=None), "null"),
    (dict(ws=None), "null"), (dict(status=None), "null"), (dict(ws_bytes=8), "workspace"), (dict(ws=ODD), "workspace"),
    (dict(logits=NINE), "aligned"),
])
def test_balance_refuses(kw, words):
    _refused(_balance(**kw), words)


def test_balance_backward_refuses():
    f = N.lib().dmoe_balance_loss_backward
    _refused(f(P, 0, 4, 8, 2, 0, None, 1, None, P, P, P, None, None), "gradient pointer")
    _refused(f(P, 0, 4, 8, 2, 5, None, 1, None, P, P, P, P, None), "mode")
    _refused(f(P, 0, 4, 8, 2, 0, None, 1, None, None, P, P, P, None), "null")


def test_wrappers_take_cuda_tensors_only():
    x = torch.zeros(4, 256)
    q = torch.zeros(4, 256, dtype=torch.float8_e4m3fn)
    s = torch.ones(4, 2)
    wq, wsc = torch.zeros(8, 256, dtype=torch.float8_e4m3fn), torch.ones(1, 2)
    for call in (lambda: N.quantize_blocks_e4m3(x), lambda: N.matmul_fp8_blocks(q, s, wq, wsc),
                 lambda: N.balance_loss(torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)),
                 lambda: N.Fp8BlockExperts(torch.zeros(1, 16, 16), torch.zeros(1, 16, 16), torch.zeros(1, 16, 16))):
        with pytest.raises(N.DMoEError):
            call()


def test_exchange_step_refuses():
    lib = N.lib()
    win = N.ep_window(1, 0, [4096], [4096], [4096], [4096], [4096])

    def call(w=win, E=2, d=256, inner=128, n=2, cap=64, hint=0, act=1, ws=P, nbytes=1 << 20, wd=P):
        return lib.dmoe_ep_expert_mlp_fp8_blocks(ctypes.byref(w) if w else None, P, P, P, P, wd, P, E, d, inner, P, P, n,
                                                 cap, hint, act, ws, nbytes, P, None)

    _refused(call(w=None), "window")
    _refused(call(w=N.ep_window(0, 0, [], [], [], [], [])), "window")
    _refused(call(act=3), "activation")
    _refused(call(d=200), "multiples of 16")
    _refused(call(inner=24), "multiples of 16")
    _refused(call(E=0), "E_stack")
    _refused(call(n=1025), "n_seg")
    _refused(call(hint=-1), "rows_hint")
    _refused(call(cap=1 << 31), "capacity")
    _refused(call(wd=None), "null")
    _refused(call(nbytes=100), "workspace")
    _refused(call(w=N.ep_window(1, 0, [4096], [4096], [4096], [4096], [4100])), "return rows")
    assert call(n=0) == 0 and call(cap=0) == 0


def test_record_bytes():
    assert [N.fp8_block_record_bytes(d) for d in (16, 256, 2064, 7168)] == [32, 272, 2064 + 80, 7168 + 224]


def test_workspace_sizes():
    lib = N.lib()
    assert lib.dmoe_grouped_mlp_fp8_blocks_workspace_size(100, 272) >= 100 * 272 + 100 * 3 * 4
    assert lib.dmoe_grouped_mlp_fp8_blocks_workspace_size(0, 272) > 0
    assert lib.dmoe_balance_loss_workspace_size() % 8 == 0


def _huge(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")  # sizes without memory


_F8, _F32, _I32, _I64 = torch.float8_e4m3fn, torch.float32, torch.int32, torch.int64
_PAST = 2**32 + 256  # what a 32-bit argument would take for 256


@pytest.mark.parametrize("call", [
    lambda: N.quantize_blocks_e4m3(_huge(1, _PAST)),
    lambda: N.quantize_blocks_e4m3(_huge(128, _PAST), 128),
    lambda: N.quantize_block_records(_huge(1, _PAST)),
    lambda: N.matmul_fp8_blocks(_huge(_PAST, 16, dtype=_F8), _huge(_PAST, 1, dtype=_F32), _huge(8, 16, dtype=_F8), _huge(1, 1, dtype=_F32)),
    lambda: N.matmul_fp8_blocks(_huge(4, 16, dtype=_F8), _huge(4, 1, dtype=_F32), _huge(_PAST, 16, dtype=_F8), _huge(_PAST // 128, 1, dtype=_F32)),
    lambda: N.matmul_fp8_blocks(_huge(4, _PAST, dtype=_F8), _huge(4, _PAST // 128, dtype=_F32), _huge(8, _PAST, dtype=_F8),
                                _huge(1, _PAST // 128, dtype=_F32)),
    lambda: N.grouped_matmul_fp8_blocks(_huge(4, 16, dtype=_F8), _huge(4, 1, dtype=_F32), _huge(_PAST, 8, 16, dtype=_F8),
                                        _huge(_PAST, 1, 1, dtype=_F32), [0], [4]),
    lambda: N.grouped_matmul_fp8_blocks(_huge(4, 16, dtype=_F8), _huge(4, 1, dtype=_F32), _huge(1, 8, 16, dtype=_F8),
                                        _huge(1, 1, 1, dtype=_F32), [0], [2**32 + 4]),
    lambda: N.grouped_matmul_fp8_blocks(_huge(4, 16, dtype=_F8), _huge(4, 1, dtype=_F32), _huge(1, 8, 16, dtype=_F8),
                                        _huge(1, 1, 1, dtype=_F32), [-2**32], [4]),
    lambda: N.grouped_matmul_fp8_blocks(_huge(4, 16, dtype=_F8), _huge(4, 1, dtype=_F32), _huge(1, 8, 16, dtype=_F8),
                                        _huge(1, 1, 1, dtype=_F32), _huge(2**32 + 1, dtype=_I32), _huge(2**32 + 1, dtype=_I32)),
    lambda: N.balance_loss(_huge(_PAST, 8, dtype=_F32), _huge(_PAST, 2, dtype=_I64)),
    lambda: N.balance_loss(_huge(4, 2**32 + 8, dtype=_F32), _huge(4, 2, dtype=_I64)),
    lambda: N.balance_loss(_huge(4, 8, dtype=_F32), _huge(4, 2**32 + 2, dtype=_I64)),
    lambda: N.balance_loss(_huge(4, 8, dtype=_F32), _huge(4, 2, dtype=_I64), seq_end=_huge(2**32 + 1, dtype=_I32)),
    lambda: N.balance_loss(_huge(4, 8, dtype=_F32), _huge(4, 2, dtype=_I64), mode=2**32),
])
def test_wrappers_refuse_sizes_past_32_bits(call, monkeypatch):
    """Sizes that the library takes as 32-bit numbers are refused before they would wrap to others."""
    monkeypatch.setattr(N, "_one_device", lambda *t: 0)
    monkeypatch.setattr(N, "_call", lambda *a: pytest.fail("a wrapped size reached the library"))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    with pytest.raises(N.DMoEError, match="2\\^"):
        call()


def test_quantize_refuses_rows_wider_than_a_grid():
    """2^26 columns of f32 are 65,536 CTAs along the row, one more than a grid's y axis has."""
    _refused(_quantize(dtype=0, rows=1, cols=1 << 26, q_ld=1 << 26, s_ld=1 << 19), "f32 columns")


def test_import_without_cuda_in_torch():
    """A torch that was built without CUDA lacks these names; the module is imported all the same."""
    names = ("_cuda_getDevice", "_cuda_getCurrentRawStream")
    code = f"import torch\nfor n in {names!r}:\n    delattr(torch._C, n)\nimport distributedmoe_b200._native"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_balance_refuses_logits_off_their_type():
    for dt, at in ((0, 4098), (1, 4099), (2, 4097)):
        _refused(_balance(logits=ctypes.c_void_p(at), dt=dt), "aligned")
        _refused(N.lib().dmoe_balance_loss_backward(P, dt, 4, 8, 2, 0, None, 1, None, P, P, P, ctypes.c_void_p(at), None), "gradient")


def test_replaced_weights_are_checked(monkeypatch):
    """Calls take the stacks' pointers as they are then, so what replaces one has to be like it."""
    monkeypatch.setattr(N, "_one_device", lambda *t: 0)

    def stack(*shape):
        return torch.zeros(*shape, dtype=_F8), torch.ones(shape[0], -(-shape[1] // 128), -(-shape[2] // 128))

    (gq, gs), (dq, ds) = stack(2, 272, 256), stack(2, 256, 272)
    ex = N.Fp8BlockExperts.from_quantized(gq, gs, gq, gs, dq, ds)
    for name, t in (("wd_scale", torch.ones(2, 2, 2)), ("wd_scale", ds.double()), ("wg_q", gq.float()), ("wu_q", gq[:1]),
                    ("wd_q", gq), ("wg_scale", torch.ones(2, 2, 3).transpose(1, 2)), ("wu_scale", gs.to("meta"))):
        if t.is_meta:
            monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1 if t.is_meta else -1)
        with pytest.raises(N.DMoEError, match=name):
            setattr(ex, name, t)
    ex.wd_scale = ds * 2
    assert torch.equal(ex.wd_scale, ds * 2) and ex._args()[5] == ex.wd_scale.data_ptr()


def test_records_of_rows_only(monkeypatch):
    monkeypatch.setattr(N, "_one_device", lambda *t: 0)
    for shape in ((256,), (2, 3, 256)):
        with pytest.raises(N.DMoEError):
            N.quantize_block_records(torch.zeros(shape))
