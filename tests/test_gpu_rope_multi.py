"""Rotary positions with several axes (rope_multi) against the definition in 64 bits.

Tolerance per output, in units of u = 2^-24 times scale * (|x_a| + |x_b|): the reduced
angle in half turns is at most 1 and rounded once (u/2, times pi: 1.6 u in radians),
sine and cosine have one ulp (1 u), their product with the scale, the two products and
the sum round once each (0.5 u + 1 u at most of what they add up): 5 u. Outputs of 16
bits add half a step of their type (and of its smallest step).
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# (relative half step, half of the smallest subnormal step): fp16 has 11 significant bits, steps of 2^-10 relative
# to the binade, half of one 2^-11; bf16 has 8, steps of 2^-7, half of one 2^-8
HALF_STEP = {"float32": (0.0, 0.0), "float16": (2.0 ** -11, 2.0 ** -25), "bfloat16": (2.0 ** -8, 0.0)}


def axes_of(sections, order, half):
    n = len(sections)
    if order == "blocks":
        one = [a for a, k in enumerate(sections) for _ in range(k)]
        return [one[i % len(one)] for i in range(half)]
    return [i % n if i // n < sections[i % n] else 0 for i in range(half)]


def reference(x, pos, inv_freq, sections, layout, order, scale):
    """(y, magnitude) in fp64 from numpy arrays: x (C, H, D), pos (axes, C), inv_freq (half)."""
    half = len(inv_freq)
    phi = pos[axes_of(sections, order, half)].astype(np.longdouble).T * inv_freq.astype(np.longdouble)
    c, s = np.cos(phi)[:, None, :].astype(np.float64), np.sin(phi)[:, None, :].astype(np.float64)
    y, mag = x.astype(np.float64).copy(), np.abs(x.astype(np.float64))
    i = np.arange(half)
    a, b = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    xa, xb = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
    y[..., a], y[..., b] = scale * (xa * c - xb * s), scale * (xb * c + xa * s)
    mag[..., a] = mag[..., b] = abs(scale) * (np.abs(xa) + np.abs(xb))
    return y, mag


def check(got, x, pos, inv_freq, sections, layout="half", order="blocks", scale=1.0):
    want, mag = reference(x, pos, inv_freq, sections, layout, order, scale)
    rel, least = HALF_STEP[str(got.dtype).replace("torch.", "")]
    g = got.double().cpu().numpy()
    tol = 5 * U * mag
    tol = tol + rel * (np.abs(want) + tol) + least
    half = len(inv_freq)
    tol[..., 2 * half:] = rel * np.abs(want[..., 2 * half:]) + least  # copied values: rounded to the type, or kept
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size}, first {np.argwhere(bad)[0]}: {g[bad][0]} for {want[bad][0]}"


def positions(rng, axes, ncols, far):
    return rng.integers(-min(far, 100), far + 1, (axes, ncols)).astype(np.int32)


def run(q4k, seed, ncols, heads, dim, n_rot, sections, layout, order, far, dtype="float32", base=1e6, scale=1.0):
    import torch
    rng = np.random.default_rng(seed)
    xs = [rng.standard_normal((ncols, h, dim)).astype(np.float32) for h in heads]
    pos = positions(rng, len(sections), ncols, far)
    inv = q4k.rope_inv_freq(n_rot, base)
    got = q4k.rope_multi([torch.from_numpy(x).cuda() for x in xs], torch.from_numpy(pos).cuda(), inv, sections,
                         layout=layout, order=order, scale=scale, dtype=getattr(torch, dtype))
    for g, x in zip(got, xs):
        check(g, x, pos, inv.cpu().numpy(), sections, layout, order, scale)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("layout", ["half", "adjacent"])
@pytest.mark.parametrize("order", ["blocks", "interleaved"])
@pytest.mark.parametrize("ncols,heads,dim,n_rot,sections", [
    (1, (32, 8), 128, 128, (16, 24, 24)), (8, (32, 8), 128, 128, (24, 20, 20)), (3, (1,), 2, 2, (1,)), (5, (7, 1), 80, 40, (5, 5, 10)),
    (17, (3,), 33, 6, (1, 2)), (2, (2, 5), 256, 256, (32, 32, 32, 32)), (65, (4, 2), 64, 64, (3, 0, 2)), (130, (5, 3), 96, 64, (12, 10, 10)),
    (300, (2,), 1024, 1022, (100, 200, 100)), (4, (3,), 20, 0, (1,)), (9, (2, 2), 128, 126, (63,)),
])
def test_rope_shapes(q4k, ncols, heads, dim, n_rot, sections, layout, order, dtype):
    run(q4k, ncols + dim, ncols, heads, dim, n_rot, sections, layout, order, 4000, dtype)


@pytest.mark.parametrize("far", [0, 1, 1000, 1 << 17, 1 << 24, (1 << 31) - 1])
def test_rope_far_positions(q4k, far):
    run(q4k, 1, 40, (4,), 128, 128, (16, 24, 24), "half", "blocks", far, base=1e4)
    run(q4k, 2, 40, (4,), 128, 128, (16, 24, 24), "half", "interleaved", far, base=5e6, scale=1.3)


def test_rope_same_positions_on_all_axes_is_one_axis(q4k):
    import torch
    x = torch.randn(6, 4, 64, device="cuda")
    p = torch.arange(100, 106, dtype=torch.int32, device="cuda")
    inv = q4k.rope_inv_freq(64)
    one = q4k.rope_multi(x, p[None], inv, (32,))
    three = q4k.rope_multi(x, p.expand(3, 6), inv, (8, 12, 12))
    assert torch.equal(one, three)


def test_rope_positions_add_up_and_zero_keeps(q4k):
    """Turning by p and then by -p (a shift of cached keys) gives the values back; position 0 changes nothing."""
    import torch
    x = torch.randn(5, 3, 128, device="cuda")
    inv = q4k.rope_inv_freq(128, 1e4)
    p = torch.randint(0, 50000, (2, 5), dtype=torch.int32, device="cuda")
    back = q4k.rope_multi(q4k.rope_multi(x, p, inv, (32, 32)), -p, inv, (32, 32))
    mag = x.abs() + torch.cat([x[..., 64:], x[..., :64]], -1).abs()
    assert ((back - x).abs() <= 2 * 5 * U * 2 * mag).all()
    assert torch.equal(q4k.rope_multi(x, torch.zeros_like(p), inv, (32, 32)), x)


@pytest.mark.parametrize("dim,n_rot", [(128, 128), (96, 64), (50, 30)])
@pytest.mark.parametrize("ncols", [4, 300])
def test_rope_strides_in_place_and_untouched_memory(q4k, dim, n_rot, ncols):
    """q and k as slices of one fused buffer, turned in place; v between the columns keeps its values."""
    import torch
    rng = np.random.default_rng(dim)
    hq, hk = 6, 2
    for extra in (0, 3):
        buf = torch.from_numpy(rng.standard_normal((ncols, (hq + 2 * hk) * dim + extra)).astype(np.float32)).cuda()
        old = buf.cpu().numpy().copy()
        q, k = (torch.as_strided(buf, (ncols, h, dim), (buf.stride(0), dim, 1), off)
                for h, off in ((hq, 0), (hk, hq * dim)))
        pos = positions(rng, 3, ncols, 5000)
        inv = q4k.rope_inv_freq(n_rot, 1e4)
        sections = (n_rot // 2 - 2, 1, 1)
        got = q4k.rope_multi([q, k], torch.from_numpy(pos).cuda(), inv, sections, out=[q, k])
        assert got[0] is q and got[1] is k
        check(q, old[:, :hq * dim].reshape(ncols, hq, dim), pos, inv.cpu().numpy(), sections)
        check(k, old[:, hq * dim:(hq + hk) * dim].reshape(ncols, hk, dim), pos, inv.cpu().numpy(), sections)
        assert np.array_equal(buf.cpu().numpy()[:, (hq + hk) * dim:], old[:, (hq + hk) * dim:])


def test_rope_head_major_output_for_a_cache(q4k):
    """Keys written as 16-bit values into a head-major cache at an offset; the other entries keep theirs."""
    import torch
    rng = np.random.default_rng(5)
    C, H, D, room = 7, 3, 64, 50
    cache = torch.full((H, room, D), 9.0, device="cuda", dtype=torch.float16)
    x = rng.standard_normal((C, H, D)).astype(np.float32)
    pos = positions(rng, 3, C, 3000)
    inv = q4k.rope_inv_freq(D, 1e4)
    out = cache[:, 20:20 + C].transpose(0, 1)
    q4k.rope_multi(torch.from_numpy(x).cuda(), torch.from_numpy(pos).cuda(), inv, (8, 12, 12), out=out)
    check(out, x, pos, inv.cpu().numpy(), (8, 12, 12))
    assert (cache[:, :20] == 9).all() and (cache[:, 20 + C:] == 9).all()


def test_rope_nonfinite_and_special_values_stay_in_their_pair(q4k):
    import torch
    x = torch.randn(3, 2, 64, device="cuda")
    p = torch.randint(1, 9, (1, 3), dtype=torch.int32, device="cuda")
    inv = q4k.rope_inv_freq(64)
    clean = q4k.rope_multi(x, p, inv, (32,))
    x[1, 0, 5] = float("nan")
    x[2, 1, 40] = float("inf")
    got = q4k.rope_multi(x, p, inv, (32,))
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[1, 0, [5, 37]] = hit[2, 1, [40, 8]] = True
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).any()


def test_rope_inv_freq_factors(q4k):
    f = q4k.rope_inv_freq(8, 100.0, 0.5, [1.0, 2.0, 4.0, 8.0]).cpu().numpy()
    assert np.allclose(f, 0.5 * 100.0 ** (-np.arange(4) / 4) / np.array([1.0, 2.0, 4.0, 8.0]), rtol=1e-15)


def test_rope_graph_follows_positions(q4k):
    import torch
    rng = np.random.default_rng(8)
    x = rng.standard_normal((8, 40, 128)).astype(np.float32)
    xd, pos = torch.from_numpy(x).cuda(), torch.zeros(3, 8, dtype=torch.int32, device="cuda")
    inv = q4k.rope_inv_freq(128, 1e6)
    q4k.rope_multi(xd, pos, inv, (16, 24, 24))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = q4k.rope_multi(xd, pos, inv, (16, 24, 24))
    for step in range(3):
        p = positions(rng, 3, 8, 100000)
        pos.copy_(torch.from_numpy(p))
        g.replay()
        check(out, x, p, inv.cpu().numpy(), (16, 24, 24))


def test_rope_empty_and_refused_calls(q4k):
    import torch
    x, p = torch.randn(3, 2, 64, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    inv = q4k.rope_inv_freq(64)
    assert q4k.rope_multi(x[:0], p[:, :0], inv, (16, 16)).shape == (0, 2, 64)
    assert q4k.rope_multi(x[:, :0], p, inv, (16, 16)).shape == (3, 0, 64)
    ok = dict(x=x, pos=p, inv_freq=inv, sections=(16, 16))
    for kw in (dict(x=x.half()), dict(x=x[:, :, ::2]), dict(x=[]), dict(x=[x] * 5), dict(pos=p.long()), dict(pos=p[:1]),
               dict(pos=p[:, :2]), dict(inv_freq=inv.float()), dict(sections=(0, 0)), dict(layout="neox"), dict(order="x"),
               dict(dtype=torch.float64), dict(out=x[:, :1]), dict(out=x[:, :, :32]), dict(pos=p.cpu()),
               dict(inv_freq=q4k.rope_inv_freq(66)), dict(x=[x, x], out=[x, x])):
        with pytest.raises(q4k.Q4KError):
            q4k.rope_multi(**{**ok, **kw})


def test_rope_sections_of_more_than_an_int_are_refused(q4k):
    """2^32 + 16 is not taken for 16 (nor 2^32 - 1 for -1)."""
    import torch
    x, p = torch.randn(3, 2, 64, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for sections in ((2**32 + 16, 16), (16, 2**32 + 16), (2**32 - 1, 32), (-1, 33), (1025, 1), (2**70, 1)):
        with pytest.raises((q4k.Q4KError, OverflowError)):
            q4k.rope_multi(x, p, q4k.rope_inv_freq(64), sections)


@pytest.mark.parametrize("layout", ["half", "adjacent"])
@pytest.mark.parametrize("ncols", [40, 700])
@pytest.mark.parametrize("base", [1e4, 1e6])
def test_rope_sines_and_cosines_hold_their_digits(q4k, layout, ncols, base):
    """Pairs (1, 0) give the cosine and the sine themselves, so small ones show an angle that was rounded to fp32
    (up to 2^-25 half turns, 9.4e-8, whatever the sine). Tolerance: one ulp of sincospif, half of one for the
    remainder's addition (a value's ulp is at most 2^-23 of it; 2 in all for a result in the next binade); the
    remainder's rounding and second power are below 1e-14, the fp64 product's two roundings at 1600 half turns
    1600 * 2^-52 * pi = 1.2e-12."""
    import torch
    rng = np.random.default_rng(ncols)
    half = 64
    x = np.zeros((ncols, 2, 2 * half), np.float32)
    x[..., :half if layout == "half" else None:1 if layout == "half" else 2] = 1.0
    pos = rng.integers(0, 5000, (1, ncols)).astype(np.int32)
    inv = q4k.rope_inv_freq(2 * half, base)
    got = q4k.rope_multi(torch.from_numpy(x).cuda(), torch.from_numpy(pos).cuda(), inv, (half,), layout=layout)
    want, _ = reference(x, pos, inv.cpu().numpy(), (half,), layout, "blocks", 1.0)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= 2 * 2.0 ** -23 * np.abs(want) + 2e-12).all(), (err / (2.0 ** -23 * np.abs(want) + 1e-12)).max()
