"""Rotary positions against the formula in 64 bits.

Tolerance of an element y of a pair (a, b): half a step of the output type, eps / 2 * |y| (and half a step of its
subnormals), plus what 32-bit arithmetic leaves: the fraction of a turn is rounded to fp32 once (2^-26 of a turn =
9.4e-8 rad), sincospif adds two units of 2^-24, the factor, two products and a sum one half unit each: below
6e-7 * scale * (|a| + |b|) in all.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def reference(x, pos, inv_freq, heads, d, interleaved, scale, inverse):
    """(y, tolerance) of one buffer, in 64 bits."""
    rows, r = x.shape[0], 2 * inv_freq.numel()
    t = x.double().reshape(rows, heads, d)
    ang = pos.double()[:, None] * inv_freq * (-1.0 if inverse else 1.0)
    c, s = (scale * torch.cos(ang))[:, None], (scale * torch.sin(ang))[:, None]
    lo = slice(0, r, 2) if interleaved else slice(0, r // 2)
    hi = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = t[..., lo], t[..., hi]
    y, slack = t.clone(), torch.zeros_like(t)
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    slack[..., lo] = slack[..., hi] = 6e-7 * scale * (a.abs() + b.abs())
    f = torch.finfo(x.dtype)
    tol = slack + f.eps / 2 * y.abs() + f.tiny * f.eps / 2
    tol[..., r:] = 0.0  # columns that pass through are the same bits
    return y.reshape(rows, -1), tol.reshape(rows, -1)


def close(got, want):
    y, tol = want
    bad = (got.double() - y).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - y).abs() - tol).max()):.3g}"


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,kv_heads,d,rot,inverse,far", [
    (1, 1, 1, 64, 64, False, 0),
    (7, 24, 24, 64, 32, False, 0),
    (5, 6, 2, 80, 40, True, 1000003),   # 8-byte vectors
    (33, 3, 1, 96, 6, False, 131072),   # single elements and pairs
    (19, 4, 1, 128, 128, True, 77),
    (4801, 2, 1, 128, 64, False, 2000000000),  # several rows to a block
    (3, 1, 2, 65, 2, False, 9),         # an odd head width
    (2, 2, 1, 512, 512, False, 12345),
])
def test_rotary_matches_formula(cuda, dtype, interleaved, rows, heads, kv_heads, d, rot, inverse, far):
    from sa3_b200 import ops

    g = torch.Generator(device=cuda).manual_seed(rows + d + rot)
    q = torch.randn(rows, heads * d, generator=g, device=cuda).to(DT[dtype])
    k = torch.randn(rows, kv_heads * d, generator=g, device=cuda).to(DT[dtype])
    f, scale = ops.rotary_frequencies(rot, device=cuda) if not inverse else ops.rotary_frequencies(
        rot, scaling="ramp", factor=8.0, original_length=4096, device=cuda)
    per = max(1, rows // 2)
    pos = torch.arange(rows, device=cuda) % per + far
    qo, ko = ops.rotary(q, f, heads=heads, head_dim=d, k=k, kv_heads=kv_heads, rows_per_batch=per, offset=far,
                        interleaved=interleaved, scale=scale, inverse=inverse)
    close(qo, reference(q, pos, f, heads, d, interleaved, scale, inverse))
    close(ko, reference(k, pos, f, kv_heads, d, interleaved, scale, inverse))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_positions_of_rows_negative_and_far(cuda, dtype):
    from sa3_b200 import ops

    pos = torch.tensor([0, -1, 2 ** 31 - 1, -2 ** 31, 5, 5, 1000000], dtype=torch.int32, device=cuda)
    q = torch.randn(7, 2 * 64, device=cuda).to(DT[dtype])
    f, s = ops.rotary_frequencies(64, device=cuda)
    close(ops.rotary(q, f, heads=2, row_pos=pos), reference(q, pos, f, 2, 64, False, s, False))


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_on_a_fused_buffer_leaves_the_rest(cuda, interleaved):
    from sa3_b200 import ops

    buf = torch.randn(37, 3 * 4 * 64, device=cuda).bfloat16()
    was = buf.clone()
    q, k = buf[:, :256], buf[:, 256:512]
    f, s = ops.rotary_frequencies(32, device=cuda)
    pos = torch.arange(37, device=cuda)
    got = ops.rotary(q, f, heads=4, k=k, kv_heads=4, interleaved=interleaved, out=q, k_out=k)
    assert got[0].data_ptr() == buf.data_ptr()
    close(buf[:, :256], reference(was[:, :256], pos, f, 4, 64, interleaved, s, False))
    close(buf[:, 256:512], reference(was[:, 256:512], pos, f, 4, 64, interleaved, s, False))
    assert torch.equal(buf[:, 512:], was[:, 512:])


@pytest.mark.parametrize("shift,ld", [(1, 133), (2, 134), (4, 136), (8, 136)])
def test_unaligned_views(cuda, shift, ld):
    from sa3_b200 import ops

    q = torch.randn(11 * ld + shift, device=cuda).half()[shift:].view(11, ld)[:, :128]
    f, s = ops.rotary_frequencies(64, device=cuda)
    pos = torch.arange(11, device=cuda)
    close(ops.rotary(q, f, heads=2), reference(q, pos, f, 2, 64, False, s, False))


def test_matches_the_fused_rotation_of_the_framework(cuda):
    """The same rotation as the table form of qk_norm_rope without its norm: both are the formula, rounded once to
    bf16; the table's fp32 angles leave 1e-6 * position."""
    from sa3_b200 import ops

    rows = 300
    x = torch.randn(rows, 4 * 64, device=cuda).bfloat16()
    f, _ = ops.rotary_frequencies(32, device=cuda)
    want = x.clone()
    gamma = torch.ones(64, device=cuda)
    ops.qk_norm_rope(want, 4, [0], [gamma], [True], 1e-6, ops.rope_table(rows, device=cuda), rows)
    normed = x.clone()
    ops.qk_norm_rope(normed, 4, [0], [gamma], [False], 1e-6)
    got = ops.rotary(normed, f, heads=4)
    # `normed` carries one more bf16 rounding of each input of a pair
    assert float((got.float() - want.float()).abs().max()) <= 3 * 2 ** -8 * float(want.float().abs().max()) * 1.5


def test_gradient_is_the_inverse_rotation(cuda):
    """<R x, y> = <x, R^T y>, and R^T R = scale^2, in fp32."""
    from sa3_b200 import ops

    x = torch.randn(50, 3 * 128, device=cuda)
    y = torch.randn(50, 3 * 128, device=cuda)
    f, _ = ops.rotary_frequencies(128, device=cuda)
    how = dict(heads=3, head_dim=128, offset=12345, interleaved=True, scale=1.5)
    rx, ry = ops.rotary(x, f, **how), ops.rotary(y, f, inverse=True, **how)
    a, b = (rx.double() * y.double()).sum(), (x.double() * ry.double()).sum()
    bound = 2 * 6e-7 * 1.5 * 2 * float((x.abs() * y.abs()).sum() + x.abs().sum() * 3)
    assert abs(float(a - b)) <= bound
    back = ops.rotary(rx, f, inverse=True, **how)
    assert float((back - 2.25 * x).abs().max()) <= 2 * 6e-7 * 2.25 * 2 * float(x.abs().max()) * 2


def test_empty_and_graph_replay(cuda):
    from sa3_b200 import ops

    f, s = ops.rotary_frequencies(64, device=cuda)
    assert ops.rotary(torch.empty(0, 128, device=cuda), f, heads=2).shape == (0, 128)
    q = torch.randn(9, 128, device=cuda)
    pos = torch.arange(9, dtype=torch.int32, device=cuda)
    out = torch.empty_like(q)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        ops.rotary(q, f, heads=2, row_pos=pos, out=out)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        ops.rotary(q, f, heads=2, row_pos=pos, out=out)
    q.copy_(torch.randn(9, 128, device=cuda))
    pos += 100
    gr.replay()
    torch.cuda.synchronize()
    close(out, reference(q, pos, f, 2, 64, False, s, False))


def test_frequencies(cuda):
    from sa3_b200 import ops

    f, s = ops.rotary_frequencies(64, device=cuda)
    lin, _ = ops.rotary_frequencies(64, scaling="linear", factor=4.0, device=cuda)
    assert s == 1.0 and torch.equal(lin * 4, f)
    base, _ = ops.rotary_frequencies(64, scaling="base", factor=4.0, device=cuda)
    assert float(base[0]) == 1.0 and math.isclose(float(f[-1] / base[-1]), 4.0, rel_tol=1e-12)
    ramp, s = ops.rotary_frequencies(64, scaling="ramp", factor=4.0, original_length=2048, device=cuda)
    assert float(ramp[0] / f[0]) == 1.0 and math.isclose(float(f[-1] / ramp[-1]), 4.0, rel_tol=1e-12)
    assert math.isclose(s, 0.1 * math.log(4.0) + 1.0)
