"""Attention to an encoder's states, forward and backward, against the formulas in 64 bits.

Tolerances, element by element. u is half a step of the 16-bit type (2^-8 bf16, 2^-11 fp16).
  out   every probability is rounded once before P V: u * (P |V|); the result once: u * |out|.
  dv    P rounded once: u * (P^T |dO|); the result: u * |dv|.
  dS    rounded once, u * |dS|; delta = rowsum(dO * out) comes from the rounded out, P * (u * sum |dO| |out|
        + its own P-rounding error u * sum |dO| (P |V|)).
        dq and dk: scale * (those, times |K| or |Q|), and the result's rounding.
  32-bit work (scores, exponentials, sums: relative 2^-20 or so of P) is taken in by a factor 1.25, and fp16's
  subnormal steps (2^-25 a probability or dS) by their sum against |V|, |dO|, |K|, |Q|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FLOOR = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def reference(q, k, v, dout, seqs, heads, kv_heads, d, scale):
    """seqs: (query rows, visible key rows) of each sequence, as index tensors. (values, tolerances) of out, lse, dq,
    dk, dv in 64 bits; rows of no sequence stay NaN."""
    u, fl = U[q.dtype], FLOOR[q.dtype]
    q, k, v = q.double(), k.double(), v.double()
    dout = None if dout is None else dout.double()
    nan = float("nan")
    out, dq = torch.full_like(q, nan), torch.full_like(q, nan)
    dk, dv = torch.full_like(k, nan), torch.full_like(v, nan)
    lse = torch.full((heads, q.shape[0]), nan, dtype=torch.float64, device=q.device)
    tol = [torch.zeros_like(x) for x in (out, dq, dk, dv)]
    for rq, rk, all_k in seqs:
        dk[all_k] = 0.0
        dv[all_k] = 0.0
        for h in range(heads):
            cq = slice(h * d, (h + 1) * d)
            hk = h // (heads // kv_heads)
            ck = slice(hk * d, (hk + 1) * d)
            if len(rk) == 0 or len(rq) == 0:
                out[rq, cq] = 0.0
                dq[rq, cq] = 0.0
                lse[h, rq] = -math.inf
                continue
            Q, K, V = q[rq, cq], k[rk, ck], v[rk, ck]
            S = scale * Q @ K.T
            P = torch.softmax(S, -1)
            O = P @ V
            out[rq, cq] = O
            lse[h, rq] = torch.logsumexp(S, -1)
            tol[0][rq, cq] = u * (P @ V.abs() + O.abs()) + fl * (1 + V.abs().sum(0))
            if dout is None:
                continue
            G = dout[rq, cq]
            dP = G @ V.T
            delta = (G * O).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            eS = u * dS.abs() + P * u * (G.abs() * (O.abs() + P @ V.abs())).sum(-1, keepdim=True) + fl
            dq[rq, cq] = scale * dS @ K
            dk[rk, ck] += scale * dS.T @ Q
            dv[rk, ck] += P.T @ G
            tol[1][rq, cq] = scale * eS @ K.abs()
            tol[2][rk, ck] += scale * eS.T @ Q.abs()
            tol[3][rk, ck] += (u * P + fl).T @ G.abs()
    for i, x in enumerate((dq, dk, dv)):
        tol[i + 1] += u * torch.nan_to_num(x).abs() + fl
    return (out, lse, dq, dk, dv), tol


def check(got, want, tol, what):
    seen = ~want.isnan()
    err = (got.double() - want)[seen].abs()
    lim = 1.25 * tol[seen] + 1e-6
    assert torch.isfinite(got[seen]).all(), what
    over = err > lim
    assert not bool(over.any()), f"{what}: {int(over.sum())} of {over.numel()} off, worst {float((err / lim).max()):.3g}x"


def check_lse(got, want):
    """fp32 scores and sums: 2^-20 of the largest score or so, 1e-5 absolute at these sizes."""
    seen = ~want.isnan()
    g, w = got.double()[seen], want[seen]
    assert torch.equal(g == -math.inf, w == -math.inf)
    fin = w != -math.inf
    assert float((g[fin] - w[fin]).abs().max() if fin.any() else 0.0) <= 1e-5 * max(1.0, float(w[fin].abs().max()) if fin.any() else 1.0)


def run_case(cuda, batch, lq, lk, heads, kv_heads, d, dtype, mask="none", packed=False, poison=True, backward=True,
             scale=None, seed=0, spread=1.0):
    from sa3_b200 import _lib, ops

    g = torch.Generator(device=cuda).manual_seed(seed + 31 * lq + 7 * lk + batch)
    dt = DT[dtype]
    lqs = [max(0, lq - (5 * b) % (lq + 1)) for b in range(batch)] if packed else [lq] * batch
    lks = [max(0, lk - (7 * (batch - 1 - b)) % (lk + 1)) for b in range(batch)] if packed else [lk] * batch
    pad = 3 if packed else 0  # rows behind the last sequence
    nq, nk = sum(lqs) + pad, sum(lks) + pad
    q = (torch.randn(nq, heads * d, generator=g, device=cuda) * spread).to(dt)
    k = torch.randn(nk, kv_heads * d, generator=g, device=cuda).to(dt)
    v = torch.randn(nk, kv_heads * d, generator=g, device=cuda).to(dt)
    dout = torch.randn(nq, heads * d, generator=g, device=cuda).to(dt)
    how = dict(heads=heads, kv_heads=kv_heads, head_dim=d, batch=batch, max_seqlen_q=lq, max_seqlen_k=lk,
               softmax_scale=scale)
    q0 = [sum(lqs[:b]) for b in range(batch + 1)]
    k0 = [sum(lks[:b]) for b in range(batch + 1)]
    if packed:
        how["cu_seqlens_q"] = torch.tensor(q0, dtype=torch.int32, device=cuda)
        how["cu_seqlens_k"] = torch.tensor(k0, dtype=torch.int32, device=cuda)
    vis = torch.ones(nk, dtype=torch.bool, device=cuda)
    vis[k0[-1]:] = False
    if mask in ("lengths", "both"):
        lens = [x - (3 * b) % (x + 1) for b, x in enumerate(lks)]
        how["k_lens"] = torch.tensor(lens, dtype=torch.int32, device=cuda)
        for b in range(batch):
            vis[k0[b] + lens[b]:k0[b + 1]] = False
    if mask in ("keys", "both"):
        m = torch.rand(nk, generator=g, device=cuda) < 0.6
        if batch > 1:
            m[k0[1]:k0[2]] = False  # nothing left for sequence 1
        how["key_mask"] = m
        vis &= m
    seqs = [(torch.arange(q0[b], q0[b + 1], device=cuda),
             torch.arange(k0[b], k0[b + 1], device=cuda)[vis[k0[b]:k0[b + 1]]],
             torch.arange(k0[b], k0[b + 1], device=cuda)) for b in range(batch)]
    (ro, rl, rdq, rdk, rdv), tol = reference(q, k, v, dout if backward else None, seqs, heads, kv_heads, d,
                                             scale or 1.0 / math.sqrt(d))
    if poison:  # hidden keys and rows of no sequence may hold anything
        k[~vis], v[~vis] = float("nan"), float("inf")
        q[q0[-1]:], dout[q0[-1]:] = float("nan"), float("nan")
    mark = 7.0
    out = torch.full((nq, heads * d), mark, device=cuda, dtype=dt)
    lse = torch.full((heads, nq), mark, device=cuda)
    got = ops.cross_attention(q, k, v, out=out, lse=lse, return_lse=True, **how)
    assert got[0] is out and got[1] is lse
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    check(out, ro, tol[0], "out")
    check_lse(lse, rl)
    assert bool((out[q0[-1]:] == mark).all()) and bool((lse[:, q0[-1]:] == mark).all())
    if not backward:
        return
    dq = torch.full_like(q, mark)
    dk, dv = torch.full_like(k, mark), torch.full_like(v, mark)
    ops.cross_attention_backward(dout, q, k, v, out, lse, dq=dq, dk=dk, dv=dv, **how)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    for name, a, w, e in (("dq", dq, rdq, tol[1]), ("dk", dk, rdk, tol[2]), ("dv", dv, rdv, tol[3])):
        check(a, w, e, name)
    assert bool((dq[q0[-1]:] == mark).all())
    assert bool((dk[k0[-1]:] == mark).all()) and bool((dv[k0[-1]:] == mark).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("batch,lq,lk,heads,kv_heads", [
    (1, 128, 64, 1, 1),
    (1, 17, 1, 1, 1),
    (2, 129, 65, 4, 2),
    (1, 300, 257, 3, 3),
    (1, 64, 1000, 8, 1),
])
def test_forward(cuda, dtype, d, batch, lq, lk, heads, kv_heads):
    run_case(cuda, batch, lq, lk, heads, kv_heads, d, dtype, backward=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("batch,lq,lk,heads,kv_heads", [
    (1, 1, 1, 1, 1),
    (1, 1, 257, 20, 20),
    (3, 1, 1000, 8, 1),
    (2, 1, 333, 16, 1),
    (5, 2, 40, 6, 2),
    (1, 4, 5003, 8, 2),
])
def test_few_rows(cuda, dtype, d, batch, lq, lk, heads, kv_heads):
    run_case(cuda, batch, lq, lk, heads, kv_heads, d, dtype, backward=False)


@pytest.mark.parametrize("mask", ["lengths", "keys", "both"])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk", [(1, 100), (3, 1), (150, 70), (40, 200)])
def test_masks_forward(cuda, mask, packed, d, lq, lk):
    run_case(cuda, 4, lq, lk, 4, 2, d, "bf16", mask=mask, packed=packed, backward=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("batch,lq,lk,heads,kv_heads", [
    (1, 64, 128, 1, 1),
    (1, 128, 64, 1, 1),
    (1, 1, 1, 1, 1),
    (2, 77, 33, 8, 2),
    (1, 300, 257, 3, 3),
    (2, 1000, 130, 2, 1),
    (1, 33, 700, 4, 4),
])
def test_backward(cuda, dtype, d, batch, lq, lk, heads, kv_heads):
    run_case(cuda, batch, lq, lk, heads, kv_heads, d, dtype)


@pytest.mark.parametrize("mask", ["none", "lengths", "keys", "both"])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk", [(2, 5), (150, 70), (70, 300)])
def test_masks_backward(cuda, mask, packed, d, lq, lk):
    run_case(cuda, 4, lq, lk, 4, 2, d, "bf16", mask=mask, packed=packed)


@pytest.mark.parametrize("mask", ["none", "lengths", "keys", "both"])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("batch,lq,lk,heads,kv_heads,d,dtype", [
    (1, 40, 5003, 4, 2, 64, "bf16"),    # query tiles that leave CTA slots empty
    (3, 33, 1500, 2, 1, 128, "fp16"),
    (1, 1, 9001, 2, 1, 128, "bf16"),    # single tokens over long keys
    (3, 2, 8300, 6, 2, 64, "fp16"),
])
def test_split_keys(cuda, mask, packed, batch, lq, lk, heads, kv_heads, d, dtype):
    run_case(cuda, batch, lq, lk, heads, kv_heads, d, dtype, mask=mask, packed=packed, backward=mask == "both")


@pytest.mark.parametrize("d", [64, 128])
def test_large_scores_move_the_reference_maximum(cuda, d):
    """Scores spread over hundreds: the running maximum moves in most tiles."""
    run_case(cuda, 1, 200, 700, 2, 1, d, "bf16", spread=30.0, backward=False)
    run_case(cuda, 1, 1, 700, 2, 1, d, "fp16", spread=30.0, backward=False)


def test_refuses_lengths_beyond_32_bits():
    """Lengths that the library's 32-bit arguments would cut are refused before the call."""
    from sa3_b200 import ops

    x = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16)
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    for kw in (dict(max_seqlen_q=2 ** 32 + 8, max_seqlen_k=8), dict(max_seqlen_q=8, max_seqlen_k=2 ** 31)):
        with pytest.raises(RuntimeError, match="2\\*\\*31"):
            ops.cross_attention(x, x, x, heads=1, cu_seqlens_q=cu, cu_seqlens_k=cu, **kw)
    with pytest.raises(RuntimeError):
        ops.cross_attention(x, x.clone(), x.clone(), heads=1, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=8,
                            max_seqlen_k=8, out=x)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk,heads", [(40, 2048, 2), (129, 1030, 3), (300, 640, 4), (33, 9000, 8), (200, 4096, 1)])
def test_parts_of_the_keys(d, lq, lk, heads):
    """Long keys for few query rows are read in parts, joined by a warp or a block a row: against fp64, with lse."""
    from sa3_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(lq + lk)
    q, k, v = (torch.randn(n, heads * d, device="cuda", generator=g).bfloat16() for n in (lq, lk, lk))
    mask = torch.rand(lk, device="cuda", generator=g) < 0.7
    mask[:lk // 2] = False  # whole parts are hidden
    o, lse = ops.cross_attention(q, k, v, heads=heads, head_dim=d, max_seqlen_q=lq, max_seqlen_k=lk, key_mask=mask,
                                 return_lse=True)
    qd, kd, vd = (t.double().view(-1, heads, d).transpose(0, 1) for t in (q, k, v))
    s = (qd @ kd.transpose(1, 2)) * d ** -0.5
    s = s.masked_fill(~mask, -math.inf)
    want_l = torch.logsumexp(s, -1)
    p = (s - want_l[..., None]).exp()
    want = (p @ vd).transpose(0, 1).reshape(lq, -1)
    # P is rounded to bf16 (2^-8 a term, against sum p|v|), O likewise; fp32 sums and exponentials: 2^-16 in all
    room = (p @ vd.abs()).transpose(0, 1).reshape(lq, -1) * (2 ** -8 + 2 ** -16) + want.abs() * 2 ** -8 * 1.01
    assert bool(((o.double() - want).abs() <= room + 1e-30).all())
    # scores: fp32 sums of d products, each partial sum at most |q||k|
    off = (qd.abs() @ kd.abs().transpose(1, 2)).amax(-1) * d ** -0.5 * d * 2 ** -24 + 2 ** -18 * (1 + want_l.abs())
    assert bool(((lse.double() - want_l).abs() <= off).all())


@pytest.mark.parametrize("d,heads,kv", [(64, 24, 24), (128, 16, 4)])
def test_order_of_packed_sequences(d, heads, kv):
    """Several rounds of items of unequal lengths: the same bits for a sequence wherever it stands in the batch, and
    among more sequences than the walk orders; sampled rows against 64 bits."""
    from sa3_b200 import ops

    lens = [(1500, 600), (1, 900), (0, 40), (1201, 1), (640, 0), (1777, 130), (900, 777), (333, 64)]
    g = torch.Generator(device="cuda").manual_seed(d)
    data = [[torch.randn(n, w * d, device="cuda", generator=g).bfloat16() for n, w in ((lq, heads), (lk, kv), (lk, kv), (lq, heads))]
            for lq, lk in lens]

    def go(order):
        q, k, v, do = (torch.cat([data[i][j] for i in order]) for j in range(4))
        cu = [torch.tensor([0] + [lens[i][j] for i in order]).cumsum(0).int().cuda() for j in range(2)]
        how = dict(heads=heads, kv_heads=kv, head_dim=d, cu_seqlens_q=cu[0], cu_seqlens_k=cu[1], max_seqlen_q=1777,
                   max_seqlen_k=900)
        o, lse = ops.cross_attention(q, k, v, return_lse=True, **how)
        dq, dk, dv = ops.cross_attention_backward(do, q, k, v, o, lse, **how)
        at, ak = cu[0].tolist(), cu[1].tolist()
        return {i: (o[at[n]:at[n + 1]], lse[:, at[n]:at[n + 1]], dq[at[n]:at[n + 1]], dk[ak[n]:ak[n + 1]], dv[ak[n]:ak[n + 1]])
                for n, i in enumerate(order)}

    want = go(list(range(8)))
    for order in ([7, 2, 5, 0, 6, 4, 1, 3], [3, 1, 4, 6, 0, 5, 2, 7]):
        got = go(order)
        for i in range(8):
            assert all(torch.equal(a, b) for a, b in zip(got[i], want[i])), (order, i)
    many = go([0, 1] + [2] * 60 + [3, 4, 5, 6, 7])
    for i in range(8):
        assert all(torch.equal(a, b) for a, b in zip(many[i][:3], want[i][:3])), i
    for i, (lq, lk) in enumerate(lens):
        if lq and lk:
            r = torch.arange(0, lq, max(1, lq // 37), device="cuda")
            q, k, v = (data[i][j].double() for j in range(3))
            q = q[r].view(-1, kv, heads // kv, d)
            k, v = k.view(lk, kv, d), v.view(lk, kv, d)
            p = torch.einsum("rhgd,khd->rhgk", q, k).mul(d ** -0.5).softmax(-1)
            o = torch.einsum("rhgk,khd->rhgd", p, v).flatten(1)
            room = torch.einsum("rhgk,khd->rhgd", p, v.abs()).flatten(1)
            # P and O each rounded once to bf16; 2^-16 for the fp32 work
            assert bool(((want[i][0][r].double() - o).abs() <= room * (2 ** -8 + 2 ** -16) + o.abs() * 2 ** -8 * 1.01).all())
        elif lq:
            assert not want[i][0].any() and bool((want[i][1] == -math.inf).all()) and not want[i][2].any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("batch", [38, 64])
def test_order_of_single_tokens(d, packed, batch):
    """One token of every sequence against long keys of unequal lengths, some of zero: the same bits wherever a sequence
    stands, and 64-bit values."""
    from sa3_b200 import ops

    kv, heads, longest = 8, 16, 1300
    g = torch.Generator(device="cuda").manual_seed(batch)
    lens = [longest, 0, 1] + [(37 * i * i + 11) % longest for i in range(batch - 3)]
    q = torch.randn(batch, heads * d, device="cuda", generator=g).bfloat16()
    k, v = (torch.randn(batch, longest, kv * d, device="cuda", generator=g).bfloat16() for _ in range(2))

    def go(order):
        how = dict(heads=heads, kv_heads=kv, head_dim=d, batch=batch, max_seqlen_q=1, max_seqlen_k=longest, return_lse=True)
        n = torch.tensor([lens[i] for i in order], dtype=torch.int32, device="cuda")
        if packed:
            cu = torch.cat([n.new_zeros(1), n.cumsum(0).int()])
            o, lse = ops.cross_attention(q[order], torch.cat([k[i, :lens[i]] for i in order]),
                                         torch.cat([v[i, :lens[i]] for i in order]), cu_seqlens_k=cu, **how)
        else:
            o, lse = ops.cross_attention(q[order], k[order].flatten(0, 1), v[order].flatten(0, 1), k_lens=n, **how)
        back = torch.empty(batch, dtype=torch.long)
        back[torch.tensor(order)] = torch.arange(batch)
        return o[back.cuda()], lse[:, back.cuda()]

    o, lse = go(list(range(batch)))
    for order in (list(range(batch))[::-1], [(7 * i + 3) % batch for i in range(batch)] if batch % 7 else [(5 * i + 3) % batch for i in range(batch)]):
        a, b = go(order)
        assert torch.equal(a, o) and torch.equal(b, lse)
    for i in range(batch):
        n = lens[i]
        if n == 0:
            assert not o[i].any() and bool((lse[:, i] == -math.inf).all())
            continue
        kk, vv = (t[i, :n].double().view(n, kv, d) for t in (k, v))
        s = torch.einsum("hgd,khd->hgk", q[i].double().view(kv, heads // kv, d), kk) * d ** -0.5
        p = s.softmax(-1)
        want = torch.einsum("hgk,khd->hgd", p, vv).flatten()
        # P and O rounded once each to bf16; 2^-16 for the fp32 work
        room = torch.einsum("hgk,khd->hgd", p, vv.abs()).flatten() * (2 ** -8 + 2 ** -16) + want.abs() * 2 ** -8 * 1.01
        assert bool(((o[i].double() - want).abs() <= room).all())
        assert bool(((lse[:, i].double() - s.logsumexp(-1).flatten()).abs() <= 2 ** -18 * (1 + s.abs().amax())).all())
