"""GPU: the generation-side operators together, under graph capture, on other streams and from two threads.

A decode step as a user writes it: fused-add norm to e4m3, a projection of the
dequantised row, rotation by three position axes, a product with the lm_head,
a draw.
"""
import threading

import pytest
import torch

import oracle
from _util import gpu

import kernels as K

pytestmark = pytest.mark.gpu


def _weights(g, hidden=256, heads=4, kv=2, dim=32, vocab=1031):
    dev = gpu()
    rnd = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    rot = K.MultiAxisRotaryEmbedding(dim, (8, 4, 4), 128).to(dev)
    return dict(norm=1 + 0.1 * rnd(hidden), qkv=rnd(hidden, (heads + kv) * dim) / hidden ** 0.5,
                head=rnd(heads * dim, vocab) / 4, rot=rot, heads=heads, kv=kv, dim=dim)


def _step(w, x, r, pos, u):
    with torch.no_grad():
        B = x.shape[0]
        q8, scale, s = K.hilda_fused_add_rms_norm_quant(x, r, w["norm"], 1e-6, 64)
        y = (q8.float().unflatten(-1, (-1, 64)) * scale[..., None]).flatten(-2)
        qkv = (y @ w["qkv"]).view(B, 1, w["heads"] + w["kv"], w["dim"]).transpose(1, 2)
        q, k = w["rot"](qkv[:, :w["heads"]], qkv[:, w["heads"]:], pos)
        logits = q.transpose(1, 2).reshape(B, -1) @ w["head"]
        ids, logp = K.hilda_sample(logits, u, 0.8, 40, 0.9, 0.01)
        return q8.view(torch.uint8), scale, s, q, k, logits, ids, logp


def _inputs(g, B=5, hidden=256):
    dev = gpu()
    return (torch.randn(B, hidden, generator=g).to(dev), torch.randn(B, hidden, generator=g).to(dev),
            torch.randint(0, 128, (3, B, 1), generator=g).to(dev), torch.rand(B, generator=g).to(dev))


def test_decode_step_against_the_definitions():
    g = torch.Generator().manual_seed(1)
    w, (x, r, pos, u) = _weights(g), _inputs(g)
    q8, scale, s, q, k, logits, ids, logp = _step(w, x, r, pos, u)
    v, want_scale, want_s = oracle.norm_quant_ref(x, w["norm"], r, group=64)
    assert torch.equal(s.cpu(), want_s)
    assert torch.allclose(scale.cpu().double(), want_scale, rtol=1e-5, atol=0)
    # the rotation of the k heads: their values before it, from the quantised row
    y = (q8.view(torch.float8_e4m3fn).cpu().double().unflatten(-1, (-1, 64)) * scale.cpu().double()[..., None]).flatten(-2)
    qkv = (y @ w["qkv"].cpu().double()).view(5, 1, 6, 32).transpose(1, 2)
    rot = w["rot"]
    want_k, _ = oracle.rope_axes_ref(qkv[:, 4:], rot.cos_cached[0], rot.sin_cached[0], pos, (8, 4, 4))
    assert torch.allclose(k.cpu().double(), want_k, rtol=0, atol=2e-3)  # (the fp32 product may run in fewer bits)
    want_ids, want_logp, _ = oracle.sample_ref(logits, u.cpu(), 0.8, 40, 0.9, 0.01)
    assert torch.equal(ids.cpu(), want_ids)
    assert torch.allclose(logp.cpu().double(), want_logp, rtol=0, atol=2e-5)


def test_graph_of_a_decode_step():
    """Captured once, replayed on new inputs with eager work between, each replay equal to the eager step. Two graphs of
    the same step live at once."""
    g = torch.Generator().manual_seed(2)
    w = _weights(g)
    sets = [_inputs(g) for _ in range(3)]
    static = [tuple(t.clone() for t in sets[0]) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(w, *static[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for inputs in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = _step(w, *inputs)
        graphs.append((graph, outs))
    for n in range(4):
        picked = [sets[n % 3], sets[(n + 1) % 3]]
        for (graph, _), inputs, new in zip(graphs, static, picked):
            for a, b in zip(inputs, new):
                a.copy_(b)
            graph.replay()
        for (_, outs), new in zip(graphs, picked):
            for i, (a, b) in enumerate(zip(outs, _step(w, *new))):
                assert torch.equal(a, b), f"replay {n}: output {i}"
        torch.cuda.synchronize()


def test_graph_of_rope_forward_and_backward():
    dev = gpu()
    g = torch.Generator().manual_seed(3)
    q = torch.randn(2, 9, 4, 32, generator=g).to(dev).transpose(1, 2).requires_grad_()
    k = torch.randn(2, 9, 2, 32, generator=g).to(dev).transpose(1, 2).requires_grad_()
    rot = K.MultiAxisRotaryEmbedding(32, (8, 4, 4), 64).to(dev)
    pos = torch.randint(0, 64, (3, 2, 9), generator=g).to(dev)
    dq, dk = torch.randn_like(q), torch.randn_like(k)

    def step():
        out = rot(q, k, pos)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, (q, k), (dq, dk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for n in range(3):
        pos.copy_(torch.randint(0, 64, (3, 2, 9), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b), f"replay {n}"


def test_other_streams_and_two_threads():
    g = torch.Generator().manual_seed(4)
    w = _weights(g)
    sets = [_inputs(g) for _ in range(2)]
    want = [[t.cpu() for t in _step(w, *s)] for s in sets]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    out = _step(w, *sets[n])
                got[n] = [t.cpu() for t in out]
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_elements_beyond_32_bit_offsets():
    """More than 2^31 elements a tensor: the last rows come out as they do alone."""
    dev, bf = gpu(), torch.bfloat16
    g = torch.Generator(device=dev).manual_seed(6)

    rows, hidden, n = 530_000, 4096, 5
    x = torch.zeros(rows, hidden, device=dev, dtype=bf)
    x[-n:] = torch.randn(n, hidden, device=dev, generator=g).to(bf)
    w = torch.randn(hidden, device=dev, generator=g).to(bf)
    assert x.numel() > 2 ** 31
    whole = K.hilda_fused_add_rms_norm_quant(x, x, w, group_size=128)
    alone = K.hilda_fused_add_rms_norm_quant(x[-n:], x[-n:], w, group_size=128)
    for a, b in zip(whole, alone):
        assert torch.equal(a[-n:].view(torch.uint8), b.view(torch.uint8))
    del x, whole

    T = 4_200_000
    q = torch.zeros(1, T, 4, 128, device=dev, dtype=bf).transpose(1, 2)
    k = torch.randn(1, T, 1, 128, device=dev, generator=g).to(bf).transpose(1, 2)
    q[:, :, -n:] = torch.randn(1, 4, n, 128, device=dev, generator=g).to(bf)
    rot = K.MultiAxisRotaryEmbedding(128, (16, 24, 24), 512).to(dev)
    pos = torch.randint(0, 512, (3, 1, T), device=dev, generator=g)
    assert q.numel() > 2 ** 31
    whole, alone = rot(q, k, pos), rot(q[:, :, -n:], k[:, :, -n:], pos[:, :, -n:])
    for a, b in zip(whole, alone):
        assert torch.equal(a[:, :, -n:], b)
    del q, k, whole

    rows, vocab = 14_200, 151936
    x = torch.zeros(rows, vocab, device=dev, dtype=bf)
    x[-n:] = (3 * torch.randn(n, vocab, device=dev, generator=g)).to(bf)
    u = torch.rand(rows, device=dev, generator=g)
    assert x.numel() > 2 ** 31
    for kw in ({}, dict(top_k=50), dict(top_p=0.9), dict(min_p=0.01)):
        whole, alone = K.hilda_sample(x, u, **kw), K.hilda_sample(x[-n:], u[-n:], **kw)
        assert torch.equal(whole[0][-n:], alone[0])
        assert torch.allclose(whole[1][-n:], alone[1], rtol=1e-5, atol=1e-5)
