"""Penalties, biases and masks on logits (logits_process).

The processed logits are a fixed sequence of IEEE fp32 operations, so they are compared
bit for bit with numpy's; the token exactly. The log-sum-exp is compared in 64 bits: each
exponential has a relative error of 2^-22 (its approximation) + 2^-22 (rounding of its
argument: |d| 2^-24 * 1.44 * 2, weighted by exp(-d) <= 0.37 / |d|), sums of positive
terms are off by 2^-24 per addition on the longest path, at most n/128 + 64 additions; the
logarithm and the final addition round once each (2^-23 |lse| and 2^-23).
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def make(seed, ncols, nvocab, hist=0, bias=0, masks=0, allow=0.5, repeats=True, spread=3.0):
    rng = np.random.default_rng(seed)
    d = dict(logits=(rng.standard_normal((ncols, nvocab)) * spread).astype(np.float32))
    if hist:
        h = rng.integers(0, nvocab, (ncols, hist)).astype(np.int32)
        if repeats:
            h[:, ::2] = h[:, ::2] % max(1, nvocab // 10)
            h[:, 1::7] = h[:, :1]
        h[rng.random((ncols, hist)) < 0.05] = -1  # others than tokens: ignored
        h[rng.random((ncols, hist)) < 0.02] = nvocab
        d["history"] = h
        d["history_len"] = rng.integers(-1, hist + 2, ncols).astype(np.int32)  # clamped
        d["penalties"] = np.stack([rng.choice([1.0, 1.1, 1.37, 0.8], ncols), rng.choice([0, 0.1, -0.3, 0.7], ncols),
                                   rng.choice([0, 0.5, -0.2], ncols)], 1).astype(np.float32)
    if bias:
        lens = rng.integers(0, bias + 1, ncols)
        off = np.zeros(ncols + 1, np.int32)
        off[1:] = np.cumsum(lens)
        n = max(1, int(off[-1]))
        tok = rng.integers(-1, nvocab + 1, n).astype(np.int32)
        val = rng.standard_normal(n).astype(np.float32) * 2
        if repeats:
            tok[::3] = tok[::3] % max(1, nvocab // 20)
        val[::31] = -np.inf
        d.update(bias_tokens=tok, bias_values=val, bias_offsets=off)
    if masks:
        words = (nvocab + 31) // 32
        d["mask"] = np.packbits(rng.random((masks, words * 32)) < allow, axis=1, bitorder="little").view(np.int32).copy()
        d["mask_rows"] = rng.integers(-1, masks + 1, ncols).astype(np.int32)
    return d


def reference(d):
    """(z, token, lse): z in the operator's fp32 operations, lse in fp64."""
    z = d["logits"].copy()
    C, V = z.shape
    with np.errstate(all="ignore"):
        for j in range(C):
            if d.get("bias_tokens") is not None:
                n = len(d["bias_tokens"])
                lo = min(max(int(d["bias_offsets"][j]), 0), n)
                hi = min(max(int(d["bias_offsets"][j + 1]), lo), n)
                sums = {}
                for t, v in zip(d["bias_tokens"][lo:hi].tolist(), d["bias_values"][lo:hi]):
                    if 0 <= t < V:
                        sums[t] = np.float32(sums.get(t, np.float32(0)) + v)
                for t, v in sums.items():
                    z[j, t] = z[j, t] + v
            if d.get("history") is not None:
                H = d["history"].shape[1]
                n = H if d.get("history_len") is None else min(max(int(d["history_len"][j]), 0), H)
                h = d["history"][j, :n]
                tok, cnt = np.unique(h[(h >= 0) & (h < V)], return_counts=True)
                r, f, p = d["penalties"][j]
                v = z[j, tok]
                v = np.where(v > 0, v / r, v * r).astype(np.float32)
                z[j, tok] = v - (cnt.astype(np.float32) * f + p)
            if d.get("mask") is not None:
                row = j if d.get("mask_rows") is None else int(d["mask_rows"][j])
                if 0 <= row < len(d["mask"]):
                    bits = np.unpackbits(d["mask"][row].view(np.uint8), bitorder="little")[:V]
                    z[j, bits == 0] = -np.inf
        token, lse = np.full(C, -1, np.int32), np.full(C, -np.inf)
        for j in range(C):
            live = np.flatnonzero(z[j] > -np.inf)
            if len(live):
                token[j] = live[np.argmax(z[j, live])]
                m = np.float64(z[j, token[j]])
                lse[j] = m if np.isinf(m) else m + np.log(np.exp(z[j, live].astype(np.float64) - m).sum())
            if np.isnan(z[j]).any():
                lse[j] = np.nan
    return z, token, lse


def device(d):
    import torch
    return {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in d.items()}


def check(got, d):
    z, token, lse = (t.cpu().numpy() for t in got)
    wz, wt, wl = reference(d)
    same = (z.view(np.int32) == wz.view(np.int32)) | (np.isnan(z) & np.isnan(wz)) | ((z == 0) & (wz == 0))
    assert same.all(), f"{(~same).sum()} values, first {np.argwhere(~same)[0]}: {z[~same][0]} for {wz[~same][0]}"
    assert np.array_equal(token, wt), (token, wt)
    fine = np.isfinite(wl)
    assert np.array_equal(lse[~fine], wl[~fine], equal_nan=True), (lse[~fine], wl[~fine])
    V = z.shape[1]
    tol = 2.0 ** -21 + (V / 128 + 64) * 2.0 ** -24 + 2.0 ** -23 * (1 + np.abs(wl[fine]))
    assert (np.abs(lse[fine] - wl[fine]) <= tol).all(), np.abs(lse[fine] - wl[fine]).max()


SHAPES = [(1, 1), (1, 31), (3, 32), (2, 33), (1, 32000), (8, 4096), (5, 4097), (8, 128256), (3, 50021), (33, 1000), (150, 8191),
          (300, 2048), (40, 128257), (700, 77)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_logits_everything_at_once(q4k, shape):
    import torch
    C, V = shape
    d = make(C + V, C, V, hist=70, bias=40, masks=max(1, C // 2))
    got = q4k.logits_process(**device(d), pick=True)
    check(got, d)
    again = q4k.logits_process(**device(d), pick=True)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("what", ["nothing", "history", "bias", "mask"])
@pytest.mark.parametrize("shape", [(2, 5000), (64, 3001)], ids=lambda s: "x".join(map(str, s)))
def test_logits_each_alone(q4k, shape, what):
    C, V = shape
    d = make(1, C, V, hist=33 * (what == "history"), bias=20 * (what == "bias"), masks=3 * (what == "mask"))
    check(q4k.logits_process(**device(d), pick=True), d)


@pytest.mark.parametrize("allow", [0.0, 0.0003, 0.01, 0.99, 1.0])
@pytest.mark.parametrize("shape", [(4, 128256), (200, 3005)], ids=lambda s: "x".join(map(str, s)))
def test_logits_mask_densities(q4k, shape, allow):
    C, V = shape
    d = make(2, C, V, hist=20, bias=10, masks=4, allow=allow)
    d["mask"][1] = 0       # allows nothing
    d["mask"][2] = 0
    d["mask"][2, -1] = 1 << ((V - 1) % 32) if (V - 1) % 32 < 31 else -(1 << 31)  # the last token only
    d["mask_rows"] = (np.arange(C) % 6 - 1).astype(np.int32)
    check(q4k.logits_process(**device(d), pick=True), d)


@pytest.mark.parametrize("hist,bias", [(1, 1), (5000, 3), (3, 3000), (20000, 4000)])
def test_logits_long_lists_and_repeats(q4k, hist, bias):
    d = make(3, 3, 40000, hist=hist, bias=bias)
    d["history_len"][:] = hist
    check(q4k.logits_process(**device(d), pick=True), d)


def test_logits_one_token_many_times(q4k):
    """The whole history and all biases on one token: the count is whole, the sum in list order."""
    d = make(4, 2, 9000, hist=4000, bias=1)
    d["history"][:] = 8999
    d["history_len"][:] = [4000, 77]
    rng = np.random.default_rng(0)
    d["bias_tokens"] = np.full(200, 8999, np.int32)
    d["bias_values"] = rng.standard_normal(200).astype(np.float32) * np.float32(10.0) ** rng.integers(-3, 4, 200).astype(np.float32)
    d["bias_offsets"] = np.array([0, 150, 200], np.int32)
    check(q4k.logits_process(**device(d), pick=True), d)


def test_logits_ties_take_the_lowest_index(q4k):
    for V in (7, 1000, 128256, 30011):
        d = dict(logits=np.zeros((4, V), np.float32))
        d["logits"][1, V // 2:] = 1.0
        d["logits"][2, V - 1] = 2.0
        d["logits"][3, [V // 3, V - 1]] = 5.0
        d["logits"][0, 0] = -0.0
        check(q4k.logits_process(**device(d), pick=True), d)


def test_logits_special_values(q4k):
    V = 6000
    d = make(6, 8, V, hist=10, bias=5, masks=2)
    lg = d["logits"]
    lg[0] = -np.inf
    lg[1, 17] = np.nan
    lg[2, 5000] = np.inf
    lg[3] = np.nan
    lg[4, :] = np.finfo(np.float32).min
    lg[5, ::2] = np.finfo(np.float32).max
    lg[6, 100] = -np.inf
    d["mask_rows"][:] = -1
    d["mask"][0] = 0
    d["mask_rows"][3] = 0  # NaN in masked places
    d["mask_rows"][7] = 0
    lg[7, 11] = np.inf
    for k in ("history_len", "bias_offsets"):
        d[k][:] = 0  # the values themselves
    check(q4k.logits_process(**device(d), pick=True), d)
    d2 = make(7, 3, V, hist=64, bias=64)
    d2["logits"][0, d2["history"][0] % V] = np.inf
    d2["logits"][1, d2["history"][1] % V] = -np.inf
    d2["logits"][2, ::3] = np.nan
    d2["history_len"][:] = 64
    check(q4k.logits_process(**device(d2), pick=True), d2)


def test_logits_bad_lists_are_clamped(q4k):
    """Offsets that run backwards or out of range, lengths out of range, rows that do not exist."""
    d = make(8, 5, 500, hist=12, bias=10, masks=2)
    n = len(d["bias_tokens"])
    d["bias_offsets"] = np.array([-5, 3, 2, n + 7, 1, 4], np.int32)
    d["history_len"] = np.array([-2147483648, 2147483647, 5, 0, 12], np.int32)
    d["history"][1, 0], d["history"][1, 1] = -2147483648, 2147483647
    d["mask_rows"] = np.array([-2147483648, 2147483647, 1, 2, 0], np.int32)
    check(q4k.logits_process(**device(d), pick=True), d)


@pytest.mark.parametrize("V,off", [(1000, 0), (1001, 0), (1000, 1), (1003, 3)])
@pytest.mark.parametrize("ncols", [3, 170])
def test_logits_strides_in_place_and_untouched_memory(q4k, ncols, V, off):
    import torch
    d = make(V + off, ncols, V, hist=9, bias=6, masks=2)
    t = device(d)
    buf = torch.full((ncols + 1, V + 4 + off), 7.0, device="cuda")
    view = buf[:ncols, off:off + V]
    view.copy_(t.pop("logits"))
    got = q4k.logits_process(view, **t, out=view, pick=True)
    check(got, d)
    assert (buf[:ncols, :off] == 7).all() and (buf[:ncols, off + V:] == 7).all() and (buf[ncols:] == 7).all()


def test_logits_optional_arguments_and_broadcasts(q4k):
    import torch
    d = make(11, 4, 700, hist=6, bias=3, masks=4)
    t = device(d)
    full = {**d, "history_len": None, "mask_rows": None}
    got = q4k.logits_process(**{**t, "history_len": None, "mask_rows": None}, pick=True)
    check(got, full)
    out = q4k.logits_process(**t)
    assert torch.equal(out, q4k.logits_process(**t, pick=True)[0])
    row = {**d, "logits": np.repeat(d["logits"][:1], 4, 0)}
    check(q4k.logits_process(**{**t, "logits": t["logits"][:1].expand(4, 700)}, pick=True), row)
    one = q4k.logits_process(t["logits"][0], pick=True)  # a single vector
    assert one[0].shape == (700,) and one[1].shape == (1,)
    assert q4k.logits_process(t["logits"][:0]).shape == (0, 700)
    z, token, lse = q4k.logits_process(t["logits"][:, :0], pick=True)
    assert z.shape == (4, 0) and (token == -1).all() and (lse == float("-inf")).all()
    none = q4k.logits_process(t["logits"], history=t["history"][:, :0], penalties=t["penalties"],
                              bias_tokens=t["bias_tokens"][:0], bias_values=t["bias_values"][:0], bias_offsets=t["bias_offsets"])
    assert torch.equal(none, t["logits"])


@pytest.mark.parametrize("ncols", [2, 200])
def test_logits_graphs_and_streams(q4k, ncols):
    """Two captured graphs replayed on two streams at once, over changing inputs."""
    import torch
    ds = [make(20 + i, ncols, 5003, hist=16, bias=8, masks=3) for i in range(2)]
    ts = [device(d) for d in ds]
    graphs, outs = [], []
    for t in ts:
        q4k.logits_process(**t, pick=True)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(q4k.logits_process(**t, pick=True))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(3):
        for d, t in zip(ds, ts):
            d["logits"] = np.roll(d["logits"], step, 1)
            d["history"] = np.roll(d["history"], 1, 0)
            t["logits"].copy_(torch.from_numpy(d["logits"]))
            t["history"].copy_(torch.from_numpy(d["history"]))
        torch.cuda.synchronize()
        for _ in range(4):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for d, o in zip(ds, outs):
            check(o, d)
    got = q4k.logits_process(**ts[0], pick=True, stream=streams[0])
    streams[0].synchronize()
    check(got, ds[0])


def test_logits_refusals_of_the_wrapper(q4k):
    import torch
    d = make(12, 3, 100, hist=4, bias=3, masks=2)
    t = device(d)
    for kw in (dict(logits=t["logits"].double()), dict(logits=t["logits"][:, ::2]), dict(history=t["history"].long()),
               dict(history=t["history"][:2]), dict(penalties=None), dict(penalties=t["penalties"][:, :2]),
               dict(history_len=t["history_len"][:1]), dict(bias_values=None), dict(bias_offsets=t["bias_offsets"][:2]),
               dict(mask=t["mask"][:, :2]), dict(mask=t["mask"].float()), dict(mask_rows=t["mask_rows"].long()),
               dict(mask=None), dict(out=t["logits"][:, :50]), dict(history=t["history"].cpu())):
        with pytest.raises(q4k.Q4KError):
            q4k.logits_process(**{**t, **kw})


@pytest.mark.parametrize("off", [0, 1, 2, 3])
@pytest.mark.parametrize("V", [20, 70001])
def test_logits_largest_ids_in_lists_are_ignored(q4k, V, off):
    """Ids up to the largest int32 (padding of some tokenizers) in histories and biases, on rows that begin at every
    offset from a 16-byte boundary: the tokens before such a row's first one have places below 0."""
    import torch
    d = make(V + off, 4, V, hist=40, bias=30)
    for k in ("history", "bias_tokens"):
        flat = d[k].reshape(-1)
        flat[::4] = 2**31 - 1
        flat[1::8] = 2**31 - 4
        flat[5::8] = -2**31
    t = device(d)
    buf = torch.empty((4, V + 8 - (V + 8) % 4), device="cuda")
    logits = buf[:, off:off + V]
    logits.copy_(t.pop("logits"))
    out = torch.empty_like(buf)[:, off:off + V]
    check(q4k.logits_process(logits, **t, out=out, pick=True), d)


def test_an_output_that_does_not_fit_is_torchs_out_of_memory(q4k):
    """A terabyte of new logits: the error that torch.empty raises, and the next call runs."""
    import torch
    row = torch.zeros(1, 1 << 18, device="cuda")
    with pytest.raises(torch.OutOfMemoryError):
        q4k.logits_process(row.expand(1 << 20, 1 << 18))
    assert torch.equal(q4k.logits_process(row), row)
