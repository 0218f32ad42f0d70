"""The rotary and cross-attention operators as they are used: strided views, streams, graphs, autograd, far offsets,
and together."""
import math

import pytest
import torch

from tests.test_cross_attention_gpu import check, reference
from tests.test_rotary_gpu import close
from tests.test_rotary_gpu import reference as rotated

pytestmark = pytest.mark.gpu


def one_sequence(n, device):
    return torch.arange(n, device=device)


def uniform(batch, lq, lk, device):
    return [(one_sequence(lq, device) + b * lq, one_sequence(lk, device) + b * lk, one_sequence(lk, device) + b * lk)
            for b in range(batch)]


@pytest.mark.parametrize("lq", [1, 70])
def test_strided_views_and_outputs(cuda, lq):
    """q in a fused projection, k and v side by side, outputs in the middle of wider buffers."""
    from sa3_b200 import ops

    B, lk, H, Hk = 2, 90, 4, 2
    proj = torch.randn(B * lq, 3 * H * 64, device=cuda).bfloat16()
    kv = torch.randn(B * lk, 2 * Hk * 64, device=cuda).bfloat16()
    q, k, v = proj[:, 256:512], kv[:, :128], kv[:, 128:]
    wide = torch.full((B * lq, 3 * H * 64), 5.0, device=cuda, dtype=torch.bfloat16)
    gkv = torch.full((B * lk, 4 * Hk * 64), 5.0, device=cuda, dtype=torch.bfloat16)
    how = dict(heads=H, kv_heads=Hk, batch=B, max_seqlen_q=lq, max_seqlen_k=lk)
    out, lse = ops.cross_attention(q, k, v, out=wide[:, :256], return_lse=True, **how)
    dout = torch.randn(B * lq, 2 * H * 64, device=cuda).bfloat16()[:, 256:]
    ops.cross_attention_backward(dout, q, k, v, out, lse, dq=wide[:, 512:], dk=gkv[:, 128:256], dv=gkv[:, 256:384], **how)
    (ro, _, rq, rk, rv), tol = reference(q, k, v, dout, uniform(B, lq, lk, cuda), H, Hk, 64, 0.125)
    check(wide[:, :256], ro, tol[0], "out")
    check(wide[:, 512:], rq, tol[1], "dq")
    check(gkv[:, 128:256], rk, tol[2], "dk")
    check(gkv[:, 256:384], rv, tol[3], "dv")
    assert bool((wide[:, 256:512] == 5).all()) and bool((gkv[:, :128] == 5).all()) and bool((gkv[:, 384:] == 5).all())


@pytest.mark.parametrize("lq,lk", [(1, 300), (1, 9000), (50, 3000), (200, 120)])
def test_same_bits_every_run_and_on_another_stream(cuda, lq, lk):
    from sa3_b200 import ops

    H, Hk = 8, 2
    q, dout = (torch.randn(lq, H * 64, device=cuda).half() for _ in range(2))
    k, v = (torch.randn(lk, Hk * 64, device=cuda).half() for _ in range(2))
    how = dict(heads=H, kv_heads=Hk, max_seqlen_q=lq, max_seqlen_k=lk)

    def once():
        o, l = ops.cross_attention(q, k, v, return_lse=True, **how)
        return (o, l, *ops.cross_attention_backward(dout, q, k, v, o, l, **how))

    first = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for st in streams:  # two at once
            with torch.cuda.stream(st):
                got.append(once())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(first, g))


def test_two_captured_graphs_replayed_in_turn_and_at_once(cuda):
    """Training steps of two sizes, each its own graph with its own workspace; inputs change between replays."""
    from sa3_b200 import ops

    def make(lq, lk, seed):
        g = torch.Generator(device=cuda).manual_seed(seed)
        t = [torch.randn(n, w, generator=g, device=cuda).bfloat16() for n, w in ((lq, 512), (lk, 128), (lk, 128), (lq, 512))]
        how = dict(heads=8, kv_heads=2, max_seqlen_q=lq, max_seqlen_k=lk)

        def step():
            o, l = ops.cross_attention(t[0], t[1], t[2], return_lse=True, **how)
            return (o, *ops.cross_attention_backward(t[3], t[0], t[1], t[2], o, l, **how))

        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            step()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            res = step()
        return t, step, gr, res

    cases = [make(300, 2000, 1), make(40, 5000, 2)]
    for t, _, _, _ in cases:
        for x in t:
            x.copy_(torch.randn(x.shape, device=cuda))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        for (_, _, gr, _), st in zip(cases, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for _, step, _, res in cases:
        assert all(torch.equal(a, b) for a, b in zip(step(), res))


@pytest.mark.parametrize("lq,lk", [(1, 40), (130, 40)])
def test_offsets_beyond_32_bits(cuda, lq, lk):
    """Rows so far apart that element offsets pass 2^31."""
    from sa3_b200 import ops

    ld = 2 ** 31 // 30 // 8 * 8
    buf = torch.zeros((lk - 1) * ld + 128, device=cuda, dtype=torch.bfloat16)
    k = buf.as_strided((lk, 64), (ld, 1))
    v = buf.as_strided((lk, 64), (ld, 1), 64)
    k.copy_(torch.randn(lk, 64, device=cuda))
    v.copy_(torch.randn(lk, 64, device=cuda))
    q, dout = (torch.randn(lq, 64, device=cuda).bfloat16() for _ in range(2))
    how = dict(heads=1, max_seqlen_q=lq, max_seqlen_k=lk)
    o, l = ops.cross_attention(q, k, v, return_lse=True, **how)
    g = ops.cross_attention_backward(dout, q, k, v, o, l, **how)
    kc, vc = k.contiguous(), v.contiguous()
    want, lw = ops.cross_attention(q, kc, vc, return_lse=True, **how)
    gw = ops.cross_attention_backward(dout, q, kc, vc, o, l, **how)
    assert torch.equal(o, want) and torch.equal(l, lw) and all(torch.equal(a, b) for a, b in zip(g, gw))
    f, s = ops.rotary_frequencies(64, device=cuda)
    pos = one_sequence(lk, cuda)
    close(ops.rotary(k, f, heads=1), rotated(kc, pos, f, 1, 64, False, s, False))
    ops.rotary(k, f, heads=1, out=k)
    close(k, rotated(kc, pos, f, 1, 64, False, s, False))


def test_many_short_sequences(cuda):
    from sa3_b200 import ops

    g = torch.Generator().manual_seed(3)
    lq = torch.randint(0, 20, (300,), generator=g).tolist()
    lk = torch.randint(0, 30, (300,), generator=g).tolist()
    cq, ck = ([0] + torch.tensor(x).cumsum(0).tolist() for x in (lq, lk))
    q = torch.randn(cq[-1], 128, device=cuda).bfloat16()
    k, v = (torch.randn(ck[-1], 64, device=cuda).bfloat16() for _ in range(2))
    how = dict(heads=2, kv_heads=1, max_seqlen_q=max(lq), max_seqlen_k=max(lk),
               cu_seqlens_q=torch.tensor(cq, dtype=torch.int32, device=cuda),
               cu_seqlens_k=torch.tensor(ck, dtype=torch.int32, device=cuda))
    out, lse = ops.cross_attention(q, k, v, return_lse=True, **how)
    dout = torch.randn_like(q)
    got = ops.cross_attention_backward(dout, q, k, v, out, lse, **how)
    seqs = [(torch.arange(cq[b], cq[b + 1], device=cuda), torch.arange(ck[b], ck[b + 1], device=cuda),
             torch.arange(ck[b], ck[b + 1], device=cuda)) for b in range(300)]
    (ro, _, *rg), tol = reference(q, k, v, dout, seqs, 2, 1, 64, 0.125)
    check(out, ro, tol[0], "out")
    for name, a, w, e in zip(("dq", "dk", "dv"), got, rg, tol[1:]):
        check(a, w, e, name)


def test_empty_tensors(cuda):
    from sa3_b200 import ops

    q = torch.randn(6, 128, device=cuda).bfloat16()
    none = torch.empty(0, 128, device=cuda, dtype=torch.bfloat16)
    how = dict(heads=2, batch=2)
    out, lse = ops.cross_attention(q, none, none, max_seqlen_q=3, return_lse=True, **how)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    dq, dk, dv = ops.cross_attention_backward(q, q, none, none, out, lse, max_seqlen_q=3, **how)
    assert bool((dq == 0).all()) and dk.shape == (0, 128) and dv.shape == (0, 128)
    big = torch.randn(2 * 40, 128, device=cuda).bfloat16()  # the tcgen05 kernel without keys
    out, lse = ops.cross_attention(big, none, none, max_seqlen_q=40, return_lse=True, **how)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    out, lse = ops.cross_attention(none, q, q, max_seqlen_k=3, return_lse=True, **how)
    assert out.shape == (0, 128) and lse.shape == (2, 0)
    dq, dk, dv = ops.cross_attention_backward(none, none, q, q, out, lse, max_seqlen_k=3, **how)
    assert bool((dk == 0).all()) and bool((dv == 0).all())


def test_refusals(cuda):
    from sa3_b200 import ops

    q = torch.randn(8, 128, device=cuda).bfloat16()
    k = torch.randn(8, 128, device=cuda).bfloat16()
    ok = dict(heads=2, max_seqlen_q=8, max_seqlen_k=8)
    out, lse = ops.cross_attention(q, k, k, return_lse=True, **ok)
    f, _ = ops.rotary_frequencies(64, device=cuda)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    bad = [
        lambda: ops.cross_attention(q.float(), k.float(), k.float(), **ok),
        lambda: ops.cross_attention(q, k.half(), k, **ok),
        lambda: ops.cross_attention(q, k, k.cpu(), **ok),
        lambda: ops.cross_attention(q, k, k[:4], **ok),
        lambda: ops.cross_attention(q, k, k, **dict(ok, max_seqlen_q=7)),
        lambda: ops.cross_attention(q, k, k, **dict(ok, heads=3)),
        lambda: ops.cross_attention(q, k, k, **dict(ok, kv_heads=1)),
        lambda: ops.cross_attention(q, k, k, head_dim=32, **dict(ok, heads=4)),
        lambda: ops.cross_attention(q.t().contiguous().t(), k, k, **ok),
        lambda: ops.cross_attention(q[:1].expand(8, 128), k, k, **ok),  # rows on top of each other
        lambda: ops.cross_attention(q, k, k, softmax_scale=0.0, **ok),
        lambda: ops.cross_attention(q, k, k, k_lens=i32(8, 8), **ok),
        lambda: ops.cross_attention(q, k, k, k_lens=torch.tensor([8], device=cuda), **ok),
        lambda: ops.cross_attention(q, k, k, key_mask=torch.ones(7, dtype=torch.bool, device=cuda), **ok),
        lambda: ops.cross_attention(q, k, k, key_mask=torch.ones(8, device=cuda), **ok),
        lambda: ops.cross_attention(q, k, k, cu_seqlens_q=i32(0, 4, 8), cu_seqlens_k=i32(0, 8), **ok),
        lambda: ops.cross_attention(q, k, k, out=torch.empty(8, 64, device=cuda, dtype=torch.bfloat16), **ok),
        lambda: ops.cross_attention(q, k, k, lse=torch.empty(8, 2, device=cuda), **ok),
        lambda: ops.cross_attention(torch.randn(8, 132, device=cuda).bfloat16()[:, 4:], k, k, **ok),
        lambda: ops.cross_attention_backward(q.float(), q, k, k, out, lse, **ok),
        lambda: ops.cross_attention_backward(q, q, k, k, out, lse[:, :4], **ok),
        lambda: ops.cross_attention_backward(q, q, k, k, out, lse, dk=torch.empty_like(q)[:4], **ok),
        lambda: ops.rotary(q, f.float(), heads=2),
        lambda: ops.rotary(q.double(), f, heads=2),
        lambda: ops.rotary(q, f, heads=3),
        lambda: ops.rotary(q, f, heads=2, k=k),
        lambda: ops.rotary(q, f, heads=2, kv_heads=2),
        lambda: ops.rotary(q, f, heads=2, k=k[:4], kv_heads=2),
        lambda: ops.rotary(q, f, heads=2, row_pos=torch.arange(8, device=cuda)),
        lambda: ops.rotary(q, f, heads=2, rows_per_batch=-1),
        lambda: ops.rotary(q, torch.cat([f, f]), heads=2),
        lambda: ops.rotary(q, f.cpu(), heads=2),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {n} was taken")


def test_autograd_matches_the_formula(cuda):
    """Rotation of queries and keys, attention with shared key heads and a mask, and back: the whole against the
    composition in 64 bits. Every rounding to 16 bits in between (rotated q and k, the gradients of both) adds half a
    step of its own to the tolerances of the single operators."""
    from sa3_b200 import autograd, ops

    torch.manual_seed(5)
    B, lq, lk, H, Hk, D = 2, 60, 45, 4, 2, 64
    dt, u = torch.float16, 2.0 ** -11
    q, k, v = (torch.randn(B * n, h * D, device=cuda).to(dt).requires_grad_() for n, h in ((lq, H), (lk, Hk), (lk, Hk)))
    mask = torch.rand(B * lk, device=cuda) < 0.7
    mask[lk:] = False  # nothing for the second sequence
    w = torch.randn(B * lq, H * D, device=cuda).to(dt)
    f, s = ops.rotary_frequencies(D, scaling="ramp", factor=4.0, original_length=1024, device=cuda)
    how = dict(heads=H, kv_heads=Hk, batch=B, max_seqlen_q=lq, max_seqlen_k=lk, key_mask=mask)
    qr = autograd.rotary(q, f, heads=H, rows_per_batch=lq, offset=1000, scale=s)
    kr = autograd.rotary(k, f, heads=Hk, rows_per_batch=lk, scale=s)
    out = autograd.cross_attention(qr, kr, v, **how)
    (out * w).sum().backward()
    seqs = [(torch.arange(lq, device=cuda) + b * lq,
             (torch.arange(lk, device=cuda) + b * lk)[mask[b * lk:(b + 1) * lk]], torch.arange(lk, device=cuda) + b * lk)
            for b in range(B)]
    # the rotated q and k as they were rounded: the rest is held to the operators' own tolerances
    pq, pk = torch.arange(B * lq, device=cuda) % lq + 1000, torch.arange(B * lk, device=cuda) % lk
    close(qr.detach(), rotated(q.detach(), pq, f, H, D, False, s, False))
    close(kr.detach(), rotated(k.detach(), pk, f, Hk, D, False, s, False))
    (ro, _, rq, rk, rv), tol = reference(qr.detach(), kr.detach(), v.detach(), w, seqs, H, Hk, D, D ** -0.5)
    check(out.detach(), ro, tol[0], "out")
    check(v.grad, rv, tol[3], "dv")
    for got, want, e, pos, heads, name in ((q.grad, rq, tol[1], pq, H, "dq"), (k.grad, rk, tol[2], pk, Hk, "dk")):
        y, _ = rotated(want, pos, f, heads, D, False, s, True)
        # the rotation back of an error: |cos| e_a + |sin| e_b <= e_a + e_b of the pair, times s, and one more rounding
        ea = e.view(-1, heads, D)
        pair = (ea[..., :D // 2] + ea[..., D // 2:]).repeat(1, 1, 2).view_as(e) * s
        check(got, y, pair + u * y.abs() + 1e-6, name)


def test_gradient_matches_differences(cuda):
    """Directional derivatives of the forward formula by central differences in 64 bits (step 1e-4, error ~1e-7 at these
    sizes) against the kernels' gradients; the tolerance is theirs, summed over the direction."""
    from sa3_b200 import ops

    torch.manual_seed(6)
    lq, lk, H, Hk, D = 20, 33, 4, 1, 128
    q, k, v, w = (torch.randn(n, h * D, device=cuda).half() for n, h in ((lq, H), (lk, Hk), (lk, Hk), (lq, H)))
    how = dict(heads=H, kv_heads=Hk, head_dim=D, max_seqlen_q=lq, max_seqlen_k=lk)
    out, lse = ops.cross_attention(q, k, v, return_lse=True, **how)
    grads = ops.cross_attention_backward(w, q, k, v, out, lse, **how)
    _, tol = reference(q, k, v, w, uniform(1, lq, lk, cuda), H, Hk, D, D ** -0.5)

    def loss(q, k, v):
        s = torch.einsum("qhd,kd->hqk", q.view(lq, H, D), k) * D ** -0.5
        return (torch.einsum("hqk,kd->qhd", torch.softmax(s, -1), v).reshape(lq, H * D) * w.double()).sum()

    x = [t.double() for t in (q, k, v)]
    for i, g in enumerate(grads):
        for _ in range(3):
            d = torch.randn_like(x[i])
            hi, lo = ([t + e * d if j == i else t for j, t in enumerate(x)] for e in (1e-4, -1e-4))
            num = float(loss(*hi) - loss(*lo)) / 2e-4
            got = float((g.double() * d).sum())
            assert abs(num - got) <= 1.25 * float((tol[i + 1] * d.abs()).sum()) + 1e-5


def test_autograd_partial_and_broadcast_gradients(cuda):
    from sa3_b200 import autograd, ops

    q = torch.randn(30, 128, device=cuda).bfloat16().requires_grad_()
    k = torch.randn(20, 128, device=cuda).bfloat16()
    how = dict(heads=2, max_seqlen_q=30, max_seqlen_k=20)
    out = autograd.cross_attention(q, k, k, **how)
    out.sum().backward()  # an expanded gradient
    o, l = ops.cross_attention(q.detach(), k, k, return_lse=True, **how)
    assert torch.equal(q.grad, ops.cross_attention_backward(torch.ones_like(o), q.detach(), k, k, o, l, **how)[0])
    f, _ = ops.rotary_frequencies(64, device=cuda)
    kk = k.clone().requires_grad_()
    a, b = autograd.rotary(q.detach()[:20], f, heads=2, k=kk, kv_heads=2)
    b.sum().backward()
    assert torch.equal(kk.grad, ops.rotary(torch.ones_like(k), f, heads=2, inverse=True))
    with torch.no_grad():
        assert torch.equal(autograd.cross_attention(q, k, k, **how), o)


def test_autograd_refuses_capture_with_gradients(cuda):
    from sa3_b200 import autograd

    q = torch.randn(30, 128, device=cuda).bfloat16().requires_grad_()
    how = dict(heads=2, max_seqlen_q=30, max_seqlen_k=30)
    autograd.cross_attention(q, q, q, **how).sum().backward()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    st = torch.cuda.Stream()
    with torch.cuda.graph(gr, stream=st):
        with pytest.raises(RuntimeError, match="captured"):
            autograd.cross_attention(q, q, q, **how)
        out = autograd.cross_attention(q.detach(), q.detach(), q.detach(), **how)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, autograd.cross_attention(q, q, q, **how))


def test_packed_autograd_leaves_zeros_behind_the_sequences(cuda):
    from sa3_b200 import autograd

    q = torch.randn(12, 128, device=cuda).bfloat16().requires_grad_()
    k = torch.randn(15, 128, device=cuda).bfloat16().requires_grad_()
    cu = torch.tensor([0, 5, 10], dtype=torch.int32, device=cuda)
    out = autograd.cross_attention(q, k, k, heads=2, max_seqlen_q=5, max_seqlen_k=5, cu_seqlens_q=cu, cu_seqlens_k=cu)
    assert bool((out[10:] == 0).all())
    out.float().square().sum().backward()
    assert bool((q.grad[10:] == 0).all()) and bool((k.grad[10:] == 0).all()) and bool(torch.isfinite(k.grad).all())
