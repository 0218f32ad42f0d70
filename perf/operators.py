"""Workloads of the rotary-position and cross-attention operators.

Four kinds of pass, each on token-row views (head h of a row in columns [h * head_dim, (h + 1) * head_dim)):

  rotary  queries and keys rotated by their positions, or (inverse) their gradients rotated back
  cross   attention of queries to an encoder's states, with grouped heads, per-sequence lengths or a key mask
  train   the same with its backward pass
  token   the same for one query token of each sequence

With ``own`` false a pass is computed by elementary torch operations; with ``own`` true by the framework's kernels.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one decoded token for each of 8 sequences, grouped heads, every position its own: the latency of a call
        dict(name="rotary_token_gqa", kind="rotary", dtype="bf16", batch=8, length=1, heads=32, kv_heads=8,
             head_dim=128, rot_dim=128, interleaved=False, inverse=False, own_pos=True, fused=False, far=131072,
             stretch=1.0),
        # the q and k streams of the medium model's fused projection (5 streams of 24 heads), both guidance halves
        dict(name="rotary_dit_medium", kind="rotary", dtype="bf16", batch=2, length=8247, heads=24, kv_heads=24,
             head_dim=64, rot_dim=32, interleaved=False, inverse=False, own_pos=False, fused=True, far=0, stretch=1.0),
        # a long prompt with interleaved pairs on half of each head and frequencies stretched for a long context
        dict(name="rotary_long_interleaved", kind="rotary", dtype="fp16", batch=1, length=40961, heads=16, kv_heads=4,
             head_dim=128, rot_dim=64, interleaved=True, inverse=False, own_pos=False, fused=False, far=500000,
             stretch=8.0),
        # the gradient of a rotation in a training step kept in 32 bits
        dict(name="rotary_grad_fp32", kind="rotary", dtype="fp32", batch=2, length=1311, heads=16, kv_heads=16,
             head_dim=64, rot_dim=32, interleaved=False, inverse=True, own_pos=True, fused=False, far=4000,
             stretch=1.0),
        # the medium model's cross-attention at its longest latent: text states of both guidance halves
        dict(name="cross_dit_medium", kind="cross", dtype="bf16", batch=2, len_q=8247, len_k=257, heads=24, kv_heads=24,
             head_dim=64, mask="none", packed=False),
        # a long prompt against long encoder states with grouped wide heads
        dict(name="cross_gqa_long", kind="cross", dtype="fp16", batch=1, len_q=4099, len_k=6001, heads=16, kv_heads=4,
             head_dim=128, mask="none", packed=False),
        # a small ragged fine-tuning batch whose key mask leaves one sequence without any key
        dict(name="train_small_masked", kind="train", dtype="fp16", batch=3, len_q=77, len_k=33, heads=8, kv_heads=2,
             head_dim=64, mask="keys", packed=False),
        # fine-tuning the medium model's cross-attention at its longest latent
        dict(name="train_dit_medium", kind="train", dtype="bf16", batch=2, len_q=8247, len_k=257, heads=24, kv_heads=24,
             head_dim=64, mask="none", packed=False),
        # packed sequences of unequal lengths, grouped wide heads
        dict(name="train_gqa_packed", kind="train", dtype="bf16", batch=4, len_q=2500, len_k=2111, heads=16, kv_heads=4,
             head_dim=128, mask="none", packed=True),
        # one token against one prompt's text states: the latency of a call
        dict(name="token_text", kind="token", dtype="bf16", batch=1, len_q=1, len_k=257, heads=24, kv_heads=24,
             head_dim=64, mask="none", packed=False),
        # a serving batch over encoder states of unequal lengths
        dict(name="token_batch_ragged", kind="token", dtype="bf16", batch=64, len_q=1, len_k=1500, heads=32, kv_heads=8,
             head_dim=128, mask="lengths", packed=False),
        # a few sequences over very long encoder states with few key heads
        dict(name="token_long", kind="token", dtype="fp16", batch=4, len_q=1, len_k=60001, heads=16, kv_heads=2,
             head_dim=128, mask="none", packed=False),
    ]


def _between(rng, lo, hi):
    """Spread over the logarithm, both ends within reach."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "cross", "train", "token"])
    dtype = rng.choice(["bf16", "fp16"])
    kv_heads = rng.choice([1, 2, 4, 8, 16, 24])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv_heads <= 32])
    if kind == "rotary":
        head_dim = rng.choice([64, 80, 96, 128])
        row = (heads + kv_heads) * head_dim
        rows = _between(rng, 1, min(40000, 10 ** 8 // row))
        batch = rng.choice([b for b in (1, 2, 3, 7, 16) if b <= rows])
        return dict(kind=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), batch=batch, length=rows // batch,
                    heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rot_dim=rng.choice([r for r in (32, 40, 64, 96, 128) if r <= head_dim]),
                    interleaved=rng.random() < 0.5, inverse=rng.random() < 0.4, own_pos=rng.random() < 0.5,
                    fused=rng.random() < 0.3, far=rng.choice([0, 5000, 131072, 1000000]),
                    stretch=rng.choice([1.0, 1.0, 4.0, 16.0]))
    head_dim = rng.choice([64, 128])
    mask = rng.choice(["none", "lengths", "keys"])
    if kind == "token":
        batch = _between(rng, 1, 96)
        most = min(60000, 10 ** 8 // (2 * batch * kv_heads * head_dim))
        return dict(kind=kind, dtype=dtype, batch=batch, len_q=1, len_k=_between(rng, 1, max(1, most)), heads=heads,
                    kv_heads=kv_heads, head_dim=head_dim, mask=mask, packed=False)
    batch = rng.choice([1, 2, 3, 5])
    most = 2 * 10 ** 10 if kind == "train" else 4 * 10 ** 10
    len_q = _between(rng, 2, 9000)
    len_k = _between(rng, 1, max(1, min(6000, most // (batch * heads * head_dim * len_q))))
    return dict(kind=kind, dtype=dtype, batch=batch, len_q=len_q, len_k=len_k, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, mask=mask, packed=rng.random() < 0.4)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(n, longest):
    """The lengths of n sequences: the first is the longest, the others spread down to a quarter of it."""
    return [longest - (b * 7919) % (3 * longest // 4 + 1) for b in range(n)]


def _seq_lengths(case):
    """(rows of queries, rows of keys, keys that may be seen) of each sequence; a key mask is not counted."""
    b, lq, lk = case["batch"], case["len_q"], case["len_k"]
    q = _lengths(b, lq) if case["packed"] else [lq] * b
    k = _lengths(b, lk)[::-1] if case["packed"] else [lk] * b
    seen = [min(x, y) for x, y in zip(k, _lengths(b, lk))] if case["mask"] == "lengths" else k
    return q, k, seen


def _offsets(lengths, device):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=device)


def _inv_freq(rot_dim, stretch):
    """Frequencies of a rotation, in 64 bits. Stretched: those that turn less than once in 4096 positions are
    divided by `stretch`, those that turn more than 32 times are kept, and a ramp joins them."""
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    f = 10000.0 ** (-i / rot_dim)
    if stretch == 1.0:
        return f
    keep = ((4096 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * keep + f / stretch * (1.0 - keep)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    s = dict(case=case)
    d = case["head_dim"]
    wq, wk = case["heads"] * d, case["kv_heads"] * d
    if case["kind"] == "rotary":
        rows = case["batch"] * case["length"]
        if case["fused"]:  # q and k side by side in the output of a fused projection, with more streams behind
            buf = randn(rows, wq + wk + 3 * wk)
            s["q"], s["k"] = buf[:, :wq], buf[:, wq:wq + wk]
        else:
            s["q"], s["k"] = randn(rows, wq), randn(rows, wk)
        s["inv_freq"] = _inv_freq(case["rot_dim"], case["stretch"]).to(dev)
        s["scale"] = 1.0 if case["stretch"] == 1.0 else 0.1 * math.log(case["stretch"]) + 1.0
        s["row_pos"] = None
        if case["own_pos"]:
            s["row_pos"] = torch.randint(0, case["far"] + case["length"], (rows,), generator=g, device=dev,
                                         dtype=torch.int32)
        return s
    lq, lk, seen = _seq_lengths(case)
    s["q"], s["k"], s["v"] = randn(sum(lq), wq), randn(sum(lk), wk), randn(sum(lk), wk)
    if case["kind"] == "train":
        s["dout"] = randn(sum(lq), wq)
    s["cu_q"] = _offsets(lq, dev) if case["packed"] else None
    s["cu_k"] = _offsets(lk, dev) if case["packed"] else None
    s["k_lens"] = torch.tensor(seen, dtype=torch.int32, device=dev) if case["mask"] == "lengths" else None
    s["key_mask"] = None
    if case["mask"] == "keys":
        m = torch.rand(sum(lk), generator=g, device=dev) < 0.8
        if case["batch"] > 1:  # the last sequence is left without any key
            m[sum(lk) - lk[-1]:] = False
        s["key_mask"] = m
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_rotary(s):
    c = s["case"]
    r, d = c["rot_dim"], c["head_dim"]
    rows = s["q"].shape[0]
    if s["row_pos"] is not None:
        pos = s["row_pos"].double()
    else:
        pos = (torch.arange(rows, device=s["q"].device) % c["length"] + c["far"]).double()
    angle = pos[:, None] * s["inv_freq"]
    cos = (torch.cos(angle) * s["scale"]).float()[:, None, :]
    sin = (torch.sin(angle) * s["scale"]).float()[:, None, :]
    if c["inverse"]:
        sin = -sin

    def one(x, heads):
        t = x.reshape(rows, heads, d).float()
        if c["interleaved"]:
            a, b = t[..., 0:r:2], t[..., 1:r:2]
        else:
            a, b = t[..., : r // 2], t[..., r // 2: r]
        u, w = a * cos - b * sin, b * cos + a * sin
        turned = torch.stack((u, w), -1).flatten(-2) if c["interleaved"] else torch.cat((u, w), -1)
        return torch.cat((turned, t[..., r:]), -1).to(x.dtype).reshape(rows, heads * d)

    return one(s["q"], c["heads"]), one(s["k"], c["kv_heads"])


def _rows(s, n, longest, cu):
    """Row indices [batch, longest] of each sequence, and which of them are its own."""
    at = torch.arange(longest, device=s["q"].device)
    b = torch.arange(n, device=s["q"].device)
    if cu is None:
        return b[:, None] * longest + at, torch.ones(n, longest, dtype=torch.bool, device=at.device)
    lens = (cu[1:] - cu[:-1]).long()
    ok = at[None, :] < lens[:, None]
    return torch.where(ok, cu[:-1].long()[:, None] + at, 0), ok


def _plain_attention(s):
    c = s["case"]
    n, lq, lk, h, hk, d = c["batch"], c["len_q"], c["len_k"], c["heads"], c["kv_heads"], c["head_dim"]
    g = h // hk
    iq, okq = _rows(s, n, lq, s["cu_q"])
    ik, see = _rows(s, n, lk, s["cu_k"])
    if s["k_lens"] is not None:
        see = see & (torch.arange(lk, device=see.device)[None, :] < s["k_lens"][:, None])
    if s["key_mask"] is not None:
        see = see & s["key_mask"][ik]
    hide = ~see[:, None, None, :]
    scale = 1.0 / math.sqrt(d)

    def queries(x):  # [n, hk, g * lq, d]
        return x[iq].float().view(n, lq, hk, g, d).permute(0, 2, 3, 1, 4).reshape(n, hk, g * lq, d)

    def keys(x):  # [n, hk, lk, d]
        return x[ik].float().view(n, lk, hk, d).transpose(1, 2)

    def query_rows(x):
        x = x.view(n, hk, g, lq, d).permute(0, 3, 1, 2, 4).reshape(n * lq, h * d)
        return x[okq.reshape(-1)]

    q, k, v = queries(s["q"]), keys(s["k"]), keys(s["v"])
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(hide, -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    o = torch.matmul(p, v)
    out = query_rows(o).to(s["q"].dtype)
    if c["kind"] != "train":
        return out
    do = queries(s["dout"])
    do = do * okq[:, None, None, :].expand(n, hk, g, lq).reshape(n, hk, g * lq, 1)
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q)
    own_k = _rows(s, n, lk, s["cu_k"])[1].reshape(-1)

    def key_rows(x):
        return x.transpose(1, 2).reshape(n * lk, hk * d)[own_k].to(s["q"].dtype)

    return out, query_rows(dq).to(s["q"].dtype), key_rows(dk), key_rows(dv)


# ------------------------------------------------------------------------------------------------ one pass
def _ops():
    at = os.path.join(os.getcwd(), "stable-audio-3_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from sa3_b200 import ops

    return ops


def run(state):
    s, c = state, state["case"]
    if c["kind"] == "rotary":
        if not own:
            return _plain_rotary(s)
        return _ops().rotary(s["q"], s["inv_freq"], k=s["k"], heads=c["heads"], kv_heads=c["kv_heads"],
                             head_dim=c["head_dim"], row_pos=s["row_pos"], rows_per_batch=c["length"],
                             offset=c["far"], interleaved=c["interleaved"], scale=s["scale"], inverse=c["inverse"])
    if not own:
        return _plain_attention(s)
    ops = _ops()
    how = dict(heads=c["heads"], kv_heads=c["kv_heads"], head_dim=c["head_dim"], batch=c["batch"],
               max_seqlen_q=c["len_q"], max_seqlen_k=c["len_k"], cu_seqlens_q=s["cu_q"], cu_seqlens_k=s["cu_k"],
               k_lens=s["k_lens"], key_mask=s["key_mask"])
    if c["kind"] != "train":
        return ops.cross_attention(s["q"], s["k"], s["v"], **how)
    out, lse = ops.cross_attention(s["q"], s["k"], s["v"], return_lse=True, **how)
    return (out, *ops.cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **how))


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "rotary":
        rows = case["batch"] * case["length"]
        return {"bytes": 2 * rows * (h + hk) * d * e + (4 * rows if case["own_pos"] else 0) + 4 * case["rot_dim"],
                "flops": 3 * rows * (h + hk) * case["rot_dim"]}
    lq, lk, seen = _seq_lengths(case)
    pairs = sum(a * b for a, b in zip(lq, seen)) * h
    q_bytes, k_bytes = sum(lq) * h * d * e, sum(seen) * hk * d * e
    if case["kind"] != "train":
        return {"bytes": 2 * q_bytes + 2 * k_bytes, "flops": 4 * pairs * d}
    return {"bytes": 4 * q_bytes + 4 * k_bytes, "flops": 14 * pairs * d}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_rotary(s):
    c = s["case"]
    r, d = c["rot_dim"], c["head_dim"]

    def one(x, heads):
        rows = x.shape[0]
        y = x.double().view(rows, heads, d).clone()
        if s["row_pos"] is None:
            p = torch.tensor([float(c["far"])], dtype=torch.float64, device=x.device) + \
                torch.arange(c["length"], dtype=torch.float64, device=x.device).repeat(c["batch"])
        else:
            p = s["row_pos"].to(torch.float64)
        turn = torch.polar(torch.full((rows, r // 2), s["scale"], dtype=torch.float64, device=x.device),
                           torch.outer(p, s["inv_freq"]) * (-1.0 if c["inverse"] else 1.0))
        lo = torch.arange(r // 2, device=x.device) * (2 if c["interleaved"] else 1)
        hi = lo + (1 if c["interleaved"] else r // 2)
        z = torch.complex(y[:, :, lo], y[:, :, hi]) * turn[:, None, :]
        y[:, :, lo], y[:, :, hi] = z.real, z.imag
        return y.view(rows, heads * d)

    return one(s["q"], c["heads"]), one(s["k"], c["kv_heads"])


def _exact_attention(s):
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    lq, lk, seen = _seq_lengths(c)
    need = c["kind"] == "train"
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    res = [torch.zeros_like(q)] + ([torch.zeros_like(x) for x in (q, k, v)] if need else [])
    for b in range(c["batch"]):
        q0, k0 = sum(lq[:b]), sum(lk[:b])
        keep = torch.arange(k0, k0 + seen[b], device=q.device)
        if s["key_mask"] is not None:
            keep = keep[s["key_mask"][k0:k0 + seen[b]]]
        if keep.numel() == 0:
            continue
        rq = slice(q0, q0 + lq[b])
        for j in range(hk):
            ck = slice(j * d, (j + 1) * d)
            kk = k[:, ck][keep].requires_grad_(need)
            vv = v[:, ck][keep].requires_grad_(need)
            for i in range(j * (h // hk), (j + 1) * (h // hk)):
                cq = slice(i * d, (i + 1) * d)
                qq = q[rq, cq].clone().requires_grad_(need)
                o = torch.softmax(torch.einsum("qd,kd->qk", qq, kk) / math.sqrt(d), -1) @ vv
                res[0][rq, cq] = o.detach()
                if need:
                    gq, gk, gv = torch.autograd.grad(o, (qq, kk, vv), s["dout"][rq, cq].double())
                    res[1][rq, cq] = gq
                    res[2][keep, ck] += gk
                    res[3][keep, ck] += gv
    return tuple(res) if need else res[0]


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rotary(s) if case["kind"] == "rotary" else _exact_attention(s)
