"""Block-scaled 8-bit experts in a layer: router, plan, gather, quantiser, gated MLP and combine as they
are used together, called one by one and inside the device-driven plane (expert_precision
"fp8_block"), against the definition in 64 bits.

Tolerance: each expert row as in the MLP's own test, rounded to bf16 (half a step, 2^-8), weighted;
the combine adds k of them in fp32 (k 2^-23) and rounds the sum to bf16 once more."""

import pytest
import torch

from test_fp8_blocks_gpu import DEV, _mlp_reference, _nat, _quantize64, _values

gpu = pytest.mark.gpu


def _weights(E, d, I, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = [(torch.randn(E, *s, generator=g, device=DEV) * 0.05).to(torch.bfloat16) for s in ((I, d), (I, d), (d, I))]
    w_r = (torch.randn(E, d, generator=g, device=DEV) * 0.05).to(torch.bfloat16)
    return w, w_r, g


def _expected(x, idx, w, weights):
    """(y, allowed error) of the layer for tokens x with experts idx [T, k] and weights w [T, k]."""
    T, k = idx.shape
    d = x.shape[1]
    y = torch.zeros(T, d, dtype=torch.float64, device=DEV)
    slack, size = torch.zeros_like(y), torch.zeros_like(y)
    q, s = _quantize64(x)
    xv = _values(q, s, 1)
    for e in range(weights[0].shape[0]):
        t, slot = torch.where(idx == e)
        if t.numel() == 0:
            continue
        g, u, dn = (_values(*_quantize64(m[e], 128), 128) for m in weights)
        rows, err = _mlp_reference(xv[t], g, u, dn, True)
        share = w[t, slot].double()[:, None]
        y.index_add_(0, t, share * rows)
        slack.index_add_(0, t, share * err)
        size.index_add_(0, t, share * (rows.abs() + err))
    slack = slack + 2.0 ** -8 * size + k * 2.0 ** -23 * size
    return y, slack + 2.0 ** -8 * (y.abs() + slack)


@gpu
@pytest.mark.parametrize("T,E,k,d,I", [(1, 8, 2, 256, 384), (5, 16, 4, 400, 272), (200, 8, 2, 512, 400), (700, 4, 2, 272, 528)])
def test_operators_one_by_one(T, E, k, d, I):
    N = _nat()
    weights, w_r, g = _weights(E, d, I, T + E)
    x = torch.randn(T, d, generator=g, device=DEV).to(torch.bfloat16)
    idx, w, _ = N.router(x, w_r, k, renormalize=True, w_dtype=torch.float32)
    plan = N.route_plan(idx, w, E)
    rows = torch.empty(T * k, d, dtype=torch.bfloat16, device=DEV)
    N.permute_rows(x, rows, [0], [0], [T * k], row_map=plan["perm_token"])
    xq, xs = N.quantize_blocks_e4m3(rows)
    Y = N.grouped_gated_mlp_fp8_blocks(xq, xs, N.Fp8BlockExperts(*weights), torch.arange(E, dtype=torch.int32, device=DEV),
                                       plan["offsets"][1:], N.ACT_SILU)
    out = torch.empty(T, d, dtype=torch.bfloat16, device=DEV)
    N.combine(Y, plan["inverse"], w, out)
    N.check_device_status(torch.device(DEV))
    want, slack = _expected(x, idx, w, weights)
    assert ((out.double() - want).abs() - slack).max().item() <= 0


@gpu
def test_records_layout():
    """Row t's codes in bytes [0, d), its scales from byte d on; a row is a multiple of 16 bytes."""
    N = _nat()
    for T, d in ((50, 256), (3, 2064), (1, 16)):
        x = torch.randn(T, d, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(torch.bfloat16)
        q, s = N.quantize_blocks_e4m3(x)
        rec = N.quantize_block_records(x)
        nb = s.shape[1]
        assert rec.shape == (T, N.fp8_block_record_bytes(d)) and rec.shape[1] % 16 == 0
        assert torch.equal(rec[:, :d], q.view(torch.uint8))
        assert torch.equal(rec[:, d:d + 4 * nb].contiguous().view(torch.float32), s)
    with pytest.raises(N.DMoEError):
        N.quantize_block_records(torch.zeros(2, 24, device=DEV))


@gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_direct_layer(graphs):
    """The device-driven plane with replicated blocks, eagerly and from captured graphs."""
    from distributedmoe_b200.MoE.local_cluster import LocalCluster
    from distributedmoe_b200.TensorTransferEngine import TensorTransferEngineBackend as B
    N = _nat()
    E, k, d, I = 8, 2, 272, 400
    weights, w_r, g = _weights(E, d, I, 23)
    blocks = [[0, 1, 2, 3], [4, 5, 6, 7], [1, 6]]
    dev = torch.device(DEV)
    cl = LocalCluster(E, blocks, k, d, torch.bfloat16, dev, [dev] * len(blocks),
                      stacked=[tuple(m[b].contiguous() for m in weights) for b in blocks], io_buffer_size=256,
                      number_of_io_buffers=1, backend=B.NVLinkDirect, max_tokens=1024, cuda_graphs=graphs,
                      expert_precision="fp8_block", activation="silu", renormalize=True)
    outs = []
    try:
        with torch.no_grad():
            cl.moe.gate.weight.copy_(w_r)
        for T in [1, 200, 1024, 200, 1]:
            x = torch.randn(T, d, generator=g, device=DEV).to(torch.bfloat16)
            outs.append((x, cl.moe(x)))
        torch.cuda.synchronize()
        N.check_device_status(dev)
    finally:
        cl.close()
    for x, y in outs:
        idx, w, _ = N.router(x, w_r, k, renormalize=True, w_dtype=torch.float32)
        want, slack = _expected(x, idx, w, weights)
        assert y.dtype == torch.bfloat16 and ((y.double() - want).abs() - slack).max().item() <= 0


@gpu
def test_direct_layer_refusals():
    from distributedmoe_b200.MoE.local_cluster import LocalCluster
    from distributedmoe_b200.TensorTransferEngine import TensorTransferEngineBackend as B
    dev = torch.device(DEV)
    for d, I, dtype, precision in ((272, 392, torch.bfloat16, "fp8_block"), (256, 384, torch.float16, "fp8_block"),
                                   (264, 384, torch.bfloat16, "fp8_block"), (256, 384, torch.bfloat16, "fp8_blocks")):
        stack = tuple(torch.zeros(2, *s, dtype=dtype, device=DEV) for s in ((I, d), (I, d), (d, I)))
        with pytest.raises(ValueError):
            LocalCluster(2, [[0, 1]], 1, d, dtype, dev, [dev], stacked=[stack], io_buffer_size=64, number_of_io_buffers=1,
                         backend=B.NVLinkDirect, max_tokens=16, expert_precision=precision)


def _codes(E, n, k, g):
    """A stack as another program may have quantised it: scales that this framework's quantiser would not
    choose (a block's largest code is not 448), values that bf16 does not hold."""
    q = (torch.randn(E, n, k, generator=g, device=DEV) * 40).clamp(-300, 300).to(torch.float8_e4m3fn)
    s = 1e-3 * (1 + torch.rand(E, -(-n // 128), -(-k // 128), generator=g, device=DEV))
    return q, s


def _expected_of(x, idx, w, values):
    """_expected for weights given as the values [E, ., .] that their codes stand for."""
    y = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    slack, size = torch.zeros_like(y), torch.zeros_like(y)
    xv = _values(*_quantize64(x), 1)
    for e in range(values[0].shape[0]):
        t, slot = torch.where(idx == e)
        if t.numel() == 0:
            continue
        rows, err = _mlp_reference(xv[t], *(m[e] for m in values), True)
        share = w[t, slot].double()[:, None]
        y.index_add_(0, t, share * rows)
        slack.index_add_(0, t, share * err)
        size.index_add_(0, t, share * (rows.abs() + err))
    slack = slack + (2.0 ** -8 + idx.shape[1] * 2.0 ** -23) * size
    return y, slack + 2.0 ** -8 * (y.abs() + slack)


def _cluster(E, blocks, k, d, stacked, **kw):
    from distributedmoe_b200.MoE.local_cluster import LocalCluster
    from distributedmoe_b200.TensorTransferEngine import TensorTransferEngineBackend as B
    dev = torch.device(DEV)
    kw = dict(dict(backend=B.NVLinkDirect, expert_precision="fp8_block"), **kw)
    return LocalCluster(E, blocks, k, d, torch.bfloat16, dev, [dev] * len(blocks), stacked=stacked, io_buffer_size=256,
                        number_of_io_buffers=1, max_tokens=512, activation="silu", renormalize=True, **kw)


@gpu
@pytest.mark.parametrize("blocks", [[[0, 1, 2, 3, 4, 5]], [[0, 1, 2], [3, 4, 5], [1, 4]]], ids=["one", "replicas"])
@pytest.mark.parametrize("graphs", [False, True])
def test_direct_layer_from_a_checkpoints_codes(blocks, graphs):
    """The layer computes on the codes it is given, without copies of them where there is one block, and
    keeps no 16-bit weights."""
    N = _nat()
    E, k, d, I = 6, 2, 272, 400
    g = torch.Generator(device=DEV).manual_seed(31)
    (gq, gs), (uq, us), (dq, ds) = _codes(E, I, d, g), _codes(E, I, d, g), _codes(E, d, I, g)
    values = [_values(q, s, 128) for q, s in ((gq, gs), (uq, us), (dq, ds))]
    w_r = (torch.randn(E, d, generator=g, device=DEV) * 0.05).to(torch.bfloat16)
    stacked = [N.Fp8BlockExperts.from_quantized(*(t.view(torch.uint8)[b].view(t.dtype) if t.dtype == gq.dtype else t[b]
                                                  for t in (gq, gs, uq, us, dq, ds))) for b in blocks]
    cl = _cluster(E, blocks, k, d, stacked, cuda_graphs=graphs)
    outs = []
    try:
        with torch.no_grad():
            cl.moe.gate.weight.copy_(w_r)
        assert cl.moe._ep["stack"] is None
        if len(blocks) == 1:
            assert cl.moe._ep["blocks"]._args() == stacked[0]._args()
        for T in (1, 300, 512, 300):
            x = torch.randn(T, d, generator=g, device=DEV).to(torch.bfloat16)
            outs.append((x, cl.moe(x)))
        torch.cuda.synchronize()
        N.check_device_status(torch.device(DEV))
    finally:
        cl.close()
    for x, y in outs:
        idx, w, _ = N.router(x, w_r, k, renormalize=True, w_dtype=torch.float32)
        want, slack = _expected_of(x, idx, w, values)
        assert ((y.double() - want).abs() - slack).max().item() <= 0


@gpu
def test_codes_where_they_do_not_belong():
    from distributedmoe_b200.TensorTransferEngine import TensorTransferEngineBackend as B
    N = _nat()
    g = torch.Generator(device=DEV).manual_seed(1)
    d, I = 256, 384
    codes = N.Fp8BlockExperts.from_quantized(*_codes(2, I, d, g), *_codes(2, I, d, g), *_codes(2, d, I, g))
    stack = tuple(torch.zeros(2, *s, dtype=torch.bfloat16, device=DEV) for s in ((I, d), (I, d), (d, I)))
    for blocks, stacked, kw in (([[0, 1]], [codes], dict(expert_precision="model")),
                                ([[0, 1]], [codes], dict(expert_precision="fp8")),
                                ([[0, 1]], [codes], dict(backend=B.NVLinkIPC)),
                                ([[0, 1], [0, 1]], [codes, stack], {})):
        with pytest.raises(ValueError, match="codes"):
            _cluster(2, blocks, 1, d, stacked, **kw)
    with pytest.raises(ValueError, match="its stack must be"):
        _cluster(3, [[0, 1, 2]], 1, d, [codes])


@gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_the_layer_keeps_the_codes_it_was_given(graphs):
    """A tensor that replaces another in the caller's stack is not the layer's: a captured graph would go on
    with the old one, which might be freed by then."""
    N = _nat()
    E, k, d, I = 4, 2, 256, 272
    g = torch.Generator(device=DEV).manual_seed(2)
    parts = [*_codes(E, I, d, g), *_codes(E, I, d, g), *_codes(E, d, I, g)]
    codes = N.Fp8BlockExperts.from_quantized(*parts)
    cl = _cluster(E, [list(range(E))], k, d, [codes], cuda_graphs=graphs)
    try:
        x = torch.randn(64, d, generator=g, device=DEV).to(torch.bfloat16)
        first = [cl.moe(x) for _ in range(3)][-1]
        codes.wd_scale = parts[5] * 2
        assert torch.equal(cl.moe(x), first)
        parts[5].mul_(2)  # values changed in place are seen
        assert torch.equal(cl.moe(x), first * 2)
        N.check_device_status(torch.device(DEV))
    finally:
        cl.close()


@gpu
def test_one_rank_of_the_sharded_cluster_from_codes():
    """The launch that puts one rank on each GPU, with one rank."""
    import socket
    from datetime import timedelta

    import torch.distributed as dist

    from distributedmoe_b200.MoE.sharded_cluster import ShardedCluster
    from distributedmoe_b200.TensorTransferEngine import TensorTransferEngineBackend as B
    N = _nat()
    E, k, d, I = 4, 2, 256, 272
    g = torch.Generator(device=DEV).manual_seed(3)
    (gq, gs), (uq, us), (dq, ds) = _codes(E, I, d, g), _codes(E, I, d, g), _codes(E, d, I, g)
    codes = N.Fp8BlockExperts.from_quantized(gq, gs, uq, us, dq, ds)
    w_r = (torch.randn(E, d, generator=g, device=DEV) * 0.05).to(torch.bfloat16)
    dev = torch.device(DEV)
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1,
                            timeout=timedelta(seconds=60))
    try:
        for bad in (dict(expert_precision="model"), dict(expert_precision="fp8_block", backend=B.NVLinkIPC)):
            with pytest.raises(ValueError, match="codes"):
                ShardedCluster(E, k, d, torch.bfloat16, dev, codes, max_tokens=256, **bad)
        cl = ShardedCluster(E, k, d, torch.bfloat16, dev, codes, activation="silu", renormalize=True, max_tokens=256,
                            expert_precision="fp8_block")
        try:
            with torch.no_grad():
                cl.moe.gate.weight.copy_(w_r)
            x = torch.randn(200, d, generator=g, device=DEV).to(torch.bfloat16)
            y = cl.moe(x)
            torch.cuda.synchronize()
            N.check_device_status(dev)
        finally:
            cl.close()
    finally:
        dist.destroy_process_group()
    idx, w, _ = N.router(x, w_r, k, renormalize=True, w_dtype=torch.float32)
    want, slack = _expected_of(x, idx, w, [_values(q, s, 128) for q, s in ((gq, gs), (uq, us), (dq, ds))])
    assert ((y.double() - want).abs() - slack).max().item() <= 0
