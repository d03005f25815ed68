"""Low-rank adapters of many requests (lora_add, lora_batch) against the definition in
64 bits.

Indexing, masks, ranks and strides are checked with small whole numbers (halves at
most): every product and partial sum is then exactly representable in fp32 (and the
adapters in fp16 and bf16), so any order of summation must give the very same bits.
Accuracy is checked on normal data: with n additions of random rounding errors of
relative size 2^-24 in the worst (serial) order, the relative 2-norm error is at most
sqrt(n) * 2^-24, n = K + rank + 1.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def make(seed, ncols, K, N, slots, rank, dtype, exact=True, ids="mixed", ragged=True):
    """Inputs on the device: x, A, B, base, ids, ranks, scales."""
    import torch
    rng = np.random.default_rng(seed)

    def values(*shape):
        if exact:
            return rng.integers(-2, 3, shape).astype(np.float32) / 2
        return rng.standard_normal(shape).astype(np.float32)

    t = getattr(torch, dtype)
    x, A, B, base = values(ncols, K), values(slots, rank, K), values(slots, N, rank), values(ncols, N)
    if exact and K > 512:  # keep sums of halves of halves far below 2^24 units
        A[:, :, rng.random(K) < 1 - 512 / K] = 0
    ranks = rng.integers(0, rank + 1, slots) if ragged else np.full(slots, rank)
    scales = rng.choice([0.5, 1.0, 2.0], slots) if exact else rng.random(slots) + 0.5
    if ids == "mixed":
        idv = rng.integers(-1, slots + 1, ncols)  # slots: out of range, no adapter
    elif ids == "none":
        idv = np.full(ncols, -1)
    elif ids == "one":
        idv = np.full(ncols, slots - 1)
    else:  # runs
        idv = np.sort(rng.integers(0, slots, ncols))
    dev = "cuda"
    return dict(x=torch.from_numpy(x).to(dev), A=torch.from_numpy(A).to(dev, t), B=torch.from_numpy(B).to(dev, t),
                base=torch.from_numpy(base).to(dev), ids=torch.from_numpy(idv.astype(np.int32)).to(dev),
                ranks=torch.from_numpy(ranks.astype(np.int32)).to(dev),
                scales=torch.from_numpy(scales.astype(np.float32)).to(dev))


def reference(d, use_base=True):
    """The definition in fp64, column by column."""
    import torch
    x, A, B = d["x"].double(), d["A"].double(), d["B"].double()
    y = d["base"].double().clone() if use_base else torch.zeros((x.shape[0], B.shape[1]), device="cuda").double()
    for j, a in enumerate(d["ids"].tolist()):
        if 0 <= a < A.shape[0]:
            r = int(d["ranks"][a]) if d.get("ranks") is not None else A.shape[1]
            s = float(d["scales"][a]) if d.get("scales") is not None else 1.0
            y[j] += s * (B[a, :, :r] @ (A[a, :r] @ x[j]))
    return y


def check_exact(got, want):
    import torch
    assert not torch.isnan(got).any()
    bad = (got.double() != want).nonzero()
    assert bad.numel() == 0, f"{bad.shape[0]} of {got.numel()} values differ, first at {bad[0].tolist()}: " \
                             f"{got[tuple(bad[0])].item()} for {want[tuple(bad[0])].item()}"


SHAPES = [  # ncols, K, N, slots, rank: one token and one value up to batches, whole tiles and ragged ones
    (1, 1, 1, 1, 1), (1, 64, 64, 2, 8), (1, 4096, 4096, 3, 16), (2, 255, 33, 3, 5), (3, 1000, 129, 2, 7), (5, 777, 1023, 4, 17),
    (8, 4096, 1024, 8, 64), (8, 14336, 512, 3, 33), (9, 512, 300, 4, 128), (13, 100, 4097, 2, 200), (17, 2048, 512, 20, 16),
    (33, 320, 72, 3, 64), (64, 1024, 2048, 7, 32), (65, 513, 257, 5, 24), (100, 96, 1100, 9, 512), (130, 2048, 640, 2, 72),
    (300, 1000, 513, 40, 24), (777, 128, 130, 6, 9), (1024, 512, 256, 3, 64), (2500, 72, 65, 1000, 4),
    (64, 48, 200, 1024, 16), (600, 40, 33, 1024, 8),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_lora_exact(q4k, shape, dtype):
    import torch
    d = make(sum(shape), *shape, dtype)
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"])
    check_exact(got, reference(d))
    again = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"])
    assert torch.equal(got, again)


@pytest.mark.parametrize("ids", ["none", "one", "runs"])
@pytest.mark.parametrize("shape", [(8, 512, 260, 3, 16), (70, 300, 129, 4, 20), (600, 256, 384, 5, 32)],
                         ids=lambda s: "x".join(map(str, s)))
def test_lora_id_patterns(q4k, shape, ids):
    d = make(7, *shape, "bfloat16", ids=ids)
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"])
    check_exact(got, reference(d))


@pytest.mark.parametrize("ncols", [3, 40, 500])
@pytest.mark.parametrize("dtype", TYPES)
def test_lora_optional_arguments(q4k, ncols, dtype):
    d = make(ncols, ncols, 200, 96, 3, 12, dtype)
    d["ranks"] = d["scales"] = None
    check_exact(q4k.lora_add(d["x"], d["A"], d["B"], d["ids"]), reference(d, use_base=False))
    check_exact(q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"]), reference(d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 4096, 4096, 2, 16), (8, 14336, 1024, 4, 64), (64, 4096, 1024, 8, 32),
                                   (512, 4096, 1024, 3, 64), (300, 1001, 515, 3, 40)], ids=lambda s: "x".join(map(str, s)))
def test_lora_accuracy(q4k, shape, dtype):
    """Normal data with a large common part, so that errors of one sign would add up."""
    import torch
    d = make(sum(shape), *shape, dtype, exact=False, ragged=False)
    d["x"] = d["x"] + 1.0
    d["base"].zero_()
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"])
    want = reference(d)
    n = shape[1] + shape[4] + 1
    err = torch.linalg.norm(got.double() - want).item()
    assert err <= n ** 0.5 * 2.0 ** -24 * torch.linalg.norm(want).item(), err


@pytest.mark.parametrize("ncols", [4, 48, 400])
def test_lora_strides_and_untouched_memory(q4k, ncols):
    """Inputs and outputs as slices of wider buffers, at odd offsets; the rest of the buffers keeps its values."""
    import torch
    K, N, slots, rank = 120, 75, 3, 10
    for off, pad in ((0, 8), (1, 3)):
        d = make(off + ncols, ncols, K, N, slots, rank, "float16")
        want = reference(d)
        xb = torch.full((ncols, K + pad + off), float("nan"), device="cuda")
        xb[:, off:off + K] = d["x"]
        Ab = torch.full((slots, rank + 1, K + pad + off), float("nan"), device="cuda", dtype=torch.float16)
        Ab[:, :rank, off:off + K] = d["A"]
        Bb = torch.full((slots, N + 2, rank + pad + off), float("nan"), device="cuda", dtype=torch.float16)
        Bb[:, :N, off:off + rank] = d["B"]
        buf = torch.full((ncols + 1, N + pad + off), 7.0, device="cuda")
        out = buf[:ncols, off:off + N]
        out.copy_(d["base"])
        q4k.lora_add(xb[:, off:off + K], Ab[:, :rank, off:off + K], Bb[:, :N, off:off + rank], d["ids"], base=out,
                     ranks=d["ranks"], scales=d["scales"], out=out)
        check_exact(out, want)
        assert (buf[:ncols, :off] == 7).all() and (buf[:ncols, off + N:] == 7).all() and (buf[ncols:] == 7).all()


@pytest.mark.parametrize("ncols", [2, 50, 300])
def test_lora_values_outside_the_rank_and_other_slots_are_not_read_into_results(q4k, ncols):
    """NaN behind a slot's rank, in slots nobody uses, and in x of columns without an adapter."""
    import torch
    d = make(ncols, ncols, 264, 90, 4, 16, "bfloat16", ids="runs")
    d["ranks"][:] = torch.tensor([0, 3, 16, 9], dtype=torch.int32)
    d["ids"][d["ids"] == 2] = 1
    d["ids"][-1] = -1
    want = reference(d)
    for a, r in enumerate([0, 3, 16, 9]):
        d["A"][a, r:] = float("nan")
        d["B"][a, :, r:] = float("nan")
    d["A"][2] = float("nan")
    d["B"][2] = float("inf")
    d["x"][-1] = float("nan")
    d["x"][d["ids"] == 0] = float("inf")  # rank 0: nothing is read
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"])
    check_exact(got, want)


@pytest.mark.parametrize("ncols", [4, 300])
def test_lora_nonfinite_inputs_stay_in_their_column(q4k, ncols):
    import torch
    d = make(3, ncols, 300, 70, 2, 8, "float16", ids="one")
    d["ranks"][:] = 8
    d["A"][1, 0, 5], d["A"][1, 1, 5] = 1.0, -1.0
    want = reference(d)
    d["x"][1, 5] = float("inf")
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"])
    rest = torch.arange(ncols, device="cuda") != 1
    check_exact(got[rest], want[rest])
    assert not torch.isfinite(got[1][(d["B"][1, :, :2] != 0).all(1)]).any()


@pytest.mark.parametrize("value", [3.0e38, 1e-38, 1e-42, 65520.0, 1e5])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ncols", [2, 260])
def test_lora_extreme_magnitudes(q4k, ncols, dtype, value):
    """One large (or tiny, or subnormal) activation against adapters of ones: the product must come through."""
    import torch
    K, N, r = 64, 32, 8
    x = torch.zeros(ncols, K, device="cuda")
    x[:, 3] = value
    t = getattr(torch, dtype)
    A, B = torch.zeros(1, r, K, device="cuda", dtype=t), torch.zeros(1, N, r, device="cuda", dtype=t)
    A[0, 2, 3] = B[0, :, 2] = 1.0
    got = q4k.lora_add(x, A, B, torch.zeros(ncols, dtype=torch.int32, device="cuda"))
    want = x[:, 3:4].expand(ncols, N)
    assert ((got.double() - want.double()).abs() <= want.double().abs() * 2.0 ** -22 + 2.0 ** -133).all(), \
        (got[0, 0].item(), want[0, 0].item())


@pytest.mark.parametrize("ncols", [8, 200])
def test_lora_batch_of_projections(q4k, ncols):
    """q, k, v (one x) and down (another x, other slots) in one call, from dicts and from a task array."""
    import torch
    shapes = [(256, 512, 4, 16), (64, 512, 4, 8), (64, 512, 4, 16), (300, 700, 9, 33)]
    ds = [make(i, ncols, K, N, s, r, "float16", ids="mixed") for i, (N, K, s, r) in enumerate(shapes)]
    for d in ds[1:]:
        d["ids"] = ds[0]["ids"]
    for d in ds[1:3]:
        d["x"] = ds[0]["x"]
    items = [dict(x=d["x"], A=d["A"], B=d["B"], base=d["base"], ranks=d["ranks"], scales=d["scales"]) for d in ds]
    for got, d in zip(q4k.lora_batch(items, ds[0]["ids"]), ds):
        check_exact(got, reference(d))
    for it, d in zip(items, ds):
        it["out"] = torch.full_like(d["base"], float("nan"))
    assert q4k.lora_batch(q4k.make_lora_tasks(items), ds[0]["ids"], ws=q4k.Workspace()) is None
    for it, d in zip(items, ds):
        check_exact(it["out"], reference(d))
    assert q4k.lora_batch([], ds[0]["ids"]) == []


@pytest.mark.parametrize("ncols", [1, 8, 150])
def test_lora_captured_graphs_follow_new_ids_and_inputs(q4k, ncols):
    """Two graphs captured without a workspace of their own, replayed on two streams at once, over changing ids."""
    import torch
    ds = [make(10 + i, ncols, 640, 384, 3, 16, "bfloat16") for i in range(2)]
    graphs, outs = [], []
    for d in ds:
        q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"],
                                     scales=d["scales"]))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(3):
        for d in ds:
            d["ids"].copy_(torch.randint(-1, 3, (ncols,), dtype=torch.int32, device="cuda"))
            d["x"].copy_(d["x"].roll(step, 1))
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for d, o in zip(ds, outs):
            check_exact(o, reference(d))


@pytest.mark.parametrize("ncols", [4, 200])
def test_lora_on_a_given_stream(q4k, ncols):
    """The stream argument, as a torch stream and as a raw handle, behind work that is still running there."""
    import torch
    d = make(5, ncols, 2048, 512, 2, 16, "float16")
    want = reference(d)
    s = torch.cuda.Stream()
    x = torch.zeros_like(d["x"])
    torch.cuda.synchronize()
    for handle in (s, s.cuda_stream):
        with torch.cuda.stream(s):
            x.zero_()
            big = torch.randn(4096, 4096, device="cuda")
            for _ in range(4):
                big = big @ big * 1e-3
            x.copy_(d["x"])
        got = q4k.lora_add(x, d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"], stream=handle)
        s.synchronize()
        check_exact(got, want)


def test_lora_beside_the_projection_it_adapts(q4k, oracle):
    """y = W x by the GEMV, then the adapters added in place behind it on the same stream."""
    import torch
    rng = np.random.default_rng(1)
    d = make(1, 4, 1024, 96, 3, 16, "float16", exact=False)
    W = q4k.gen_q4k_numpy(rng, 96, 1024)
    Wd = torch.from_numpy(W).cuda()
    for _ in range(3):  # launches follow one another closely: the second sees the first's rows
        y = q4k.mul_mat_vec_q(Wd, d["x"])
        q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=y, ranks=d["ranks"], scales=d["scales"], out=y)
    d["base"] = torch.from_numpy(oracle.gemv_f32(W, d["x"].cpu().numpy())).cuda()
    want = reference(d)
    # the GEMV's bar, and the adapter's fp32 sums: n additions of terms up to the sum of magnitudes
    mag = reference({**d, "x": d["x"].abs(), "A": d["A"].abs(), "B": d["B"].abs(), "base": d["base"].abs()})
    assert ((y.double() - want).abs() <= 1e-4 + 1e-5 * want.abs() + 1041 ** 0.5 * 2.0 ** -24 * mag).all()


@pytest.mark.parametrize("ncols", [24, 64, 700])
@pytest.mark.parametrize("dtype", TYPES)
def test_lora_gives_the_same_bits_every_time(q4k, ncols, dtype):
    """Repeated calls agree bit for bit, and a column's result does not depend on the columns beside it
    within the same launch path."""
    import torch
    d = make(ncols, ncols, 1000, 384, 5, 40, dtype, exact=False)
    run = lambda x, ids: q4k.lora_add(x, d["A"], d["B"], ids, ranks=d["ranks"], scales=d["scales"])  # noqa: E731
    first = run(d["x"], d["ids"])
    for _ in range(5):
        assert torch.equal(run(d["x"], d["ids"]), first)
    perm = torch.randperm(ncols, device="cuda")
    assert torch.equal(run(d["x"][perm], d["ids"][perm]), first[perm])


@pytest.mark.parametrize("ncols", [3, 100])
def test_lora_nothing_to_add(q4k, ncols):
    """No ranks, no slots, no K, ranks of 0 in use: dst is base, x and the adapters are not read."""
    import torch
    d = make(2, ncols, 64, 45, 3, 8, "float16")
    nan = torch.full_like(d["x"], float("nan"))
    for kw in (dict(A=d["A"][:, :0], B=d["B"][:, :, :0]), dict(A=d["A"][:0], B=d["B"][:0]),
               dict(x=d["x"][:, :0], A=d["A"][:, :, :0], B=d["B"]),
               dict(x=nan, A=d["A"], B=d["B"], ranks=torch.zeros(3, dtype=torch.int32, device="cuda"))):
        x = kw.pop("x", d["x"])
        assert torch.equal(q4k.lora_add(x, ids=d["ids"], base=d["base"], **kw), d["base"])
        assert (q4k.lora_add(x, ids=d["ids"], **kw) == 0).all()


def test_lora_workspace_of_the_caller_reports_ok(q4k):
    """Many columns in a caller's workspace with any contents: the call leaves its status word at 0."""
    import torch
    d = make(9, 200, 256, 96, 3, 8, "float16")
    ws = q4k.Workspace(1 << 20)
    ws.buf.fill_(255)
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"], ws=ws)
    check_exact(got, reference(d))
    assert ws.status() == 0
    big = make(10, 3000, 256, 96, 3, 8, "float16")  # grows on demand
    got = q4k.lora_add(big["x"], big["A"], big["B"], big["ids"], base=big["base"], ranks=big["ranks"], scales=big["scales"], ws=ws)
    check_exact(got, reference(big))
    assert ws.status() == 0


def test_lora_empty_calls(q4k):
    import torch
    d = make(2, 3, 64, 32, 2, 4, "float16")
    assert q4k.lora_add(d["x"][:0], d["A"], d["B"], d["ids"][:0]).shape == (0, 32)
    none = q4k.lora_add(d["x"], d["A"][:, :0], d["B"][:, :, :0], d["ids"], base=d["base"])
    assert torch.equal(none, d["base"])
    assert torch.equal(q4k.lora_add(d["x"], d["A"][:0], d["B"][:0], d["ids"], base=d["base"]), d["base"])
    assert torch.equal(q4k.lora_add(d["x"][:, :0], d["A"][:, :, :0], d["B"], d["ids"], base=d["base"]), d["base"])
    assert q4k.lora_add(d["x"], d["A"], d["B"][:, :0], d["ids"]).shape == (3, 0)
    assert (q4k.lora_add(d["x"], d["A"], d["B"], torch.full_like(d["ids"], -1)) == 0).all()


def test_lora_refusals_of_the_wrapper(q4k):
    import torch
    d = make(2, 3, 64, 32, 2, 4, "float16")
    ok = dict(x=d["x"], A=d["A"], B=d["B"], ids=d["ids"])
    for kw in (dict(x=d["x"].double()), dict(x=d["x"][:, :63]), dict(A=d["A"].float()), dict(A=d["A"].to(torch.int16)),
               dict(B=d["B"][:1]), dict(ids=d["ids"].long()), dict(ids=d["ids"][:2]), dict(ranks=d["ranks"][:1]),
               dict(scales=d["scales"].double()), dict(base=d["base"][:, :31]), dict(out=d["base"].double()),
               dict(A=d["A"].transpose(1, 2)), dict(x=d["x"].cpu()), dict(ids=d["ids"].cpu()), dict(out=d["x"][:, :32])):
        with pytest.raises(q4k.Q4KError):
            q4k.lora_add(**{**ok, **kw})


@pytest.mark.parametrize("ncols", [8, 100])
def test_lora_task_array_wants_its_own_number_of_columns(q4k, ncols):
    """More or fewer ids than the tensors behind a task array have columns are refused, and nothing is written."""
    import torch
    d = make(4, ncols, 64, 32, 2, 4, "float16")
    out = torch.full_like(d["base"], 7.0)
    arr = q4k.make_lora_tasks([dict(x=d["x"], A=d["A"], B=d["B"], ranks=d["ranks"], scales=d["scales"], base=d["base"], out=out)])
    for ids in (torch.cat([d["ids"], d["ids"]]), d["ids"][:-1], d["ids"][:0], d["ids"].cpu(), d["ids"].long(), d["ids"][None], None):
        with pytest.raises(q4k.Q4KError):
            q4k.lora_batch(arr, ids)
    assert (out == 7).all()
    q4k.lora_batch(arr, d["ids"])
    check_exact(out, reference(d))


def test_lora_workspace_of_another_device_is_refused(q4k):
    import torch
    d = make(4, 100, 64, 32, 2, 4, "float16")
    with pytest.raises(q4k.Q4KError, match="workspace"):
        q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], ws=q4k.Workspace(1 << 20, device="cpu"))
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], ranks=d["ranks"], scales=d["scales"], ws=q4k.Workspace(0, device="cuda"))
    check_exact(got, reference(d, use_base=False))


@pytest.mark.parametrize("where", ["x", "A", "B", "all", "nan", "base"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(8, 300, 70, 2, 24), (64, 130, 33, 3, 72), (65, 300, 140, 2, 24), (300, 257, 300, 3, 72), (200, 640, 130, 2, 130)],
                         ids=lambda s: "x".join(map(str, s)))
def test_lora_infinite_values_follow_the_definition(q4k, shape, dtype, where):
    """Infinities in x, A, B and base give the infinities (and inf - inf, 0 * inf: the NaN) of the definition, whatever
    the number of columns, and every other value is exact."""
    import torch
    ncols, K, N, slots, rank = shape
    d = make(sum(shape), *shape, dtype, ids="runs", ragged=False)
    g = torch.Generator().manual_seed(1)

    def put(t, n, value):
        flat = t.view(-1)
        at = torch.randperm(flat.numel(), generator=g)[:n].to(t.device)
        flat[at] = (torch.randint(0, 2, (n,), generator=g) * 2 - 1).to(t.device, t.dtype) * value
    d["A"][d["A"] == 0] = 0.5  # few products 0 * inf, so that most of what is hit is infinite
    d["B"][:, ::2][d["B"][:, ::2] == 0] = -0.5
    inf = float("inf")
    if where in ("x", "all"):
        put(d["x"], max(1, ncols // 8), inf)
    if where in ("A", "all"):
        put(d["A"], 2, inf)
    if where in ("B", "all"):
        put(d["B"], 5, inf)
    if where == "nan":
        put(d["x"], 2, float("nan"))
        put(d["B"], 2, float("nan"))
    if where == "base":
        put(d["base"], 20, inf)
    # term by term: a library's products may skip what they hold for zero
    x, A, B = d["x"].double(), d["A"].double(), d["B"].double()
    want = d["base"].double().clone()
    for j, a in enumerate(d["ids"].tolist()):
        if 0 <= a < slots:
            want[j] += float(d["scales"][a]) * (B[a] * (A[a] * x[j]).sum(1)).sum(1)
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"])
    bad = ~((got.double() == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{bad.sum()} of {bad.numel()}, first {bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]}"


@pytest.mark.parametrize("dtype", TYPES)
def test_lora_largest_values_of_many_columns(q4k, dtype):
    """The largest fp32 activations, and sums that overflow, in place over the base."""
    import torch
    big = torch.finfo(torch.float32).max
    ncols, K, N, r = 130, 96, 200, 16
    t = getattr(torch, dtype)
    x = torch.zeros(ncols, K, device="cuda")
    x[:, 5] = big
    x[1::2, 7] = big
    A, B = torch.zeros(1, r, K, device="cuda", dtype=t), torch.zeros(1, N, r, device="cuda", dtype=t)
    A[0, 3, 5] = A[0, 3, 7] = 1.0
    B[0, :, 3] = torch.where(torch.arange(N) % 3 == 0, -1.0, 1.0).to(t)
    B[0, 1::2, 4] = 2.0  # meets a u of 0
    y = torch.ones(ncols, N, device="cuda")
    q4k.lora_add(x, A, B, torch.zeros(ncols, dtype=torch.int32, device="cuda"), base=y, out=y)
    u = torch.where(torch.arange(ncols, device="cuda") % 2 == 1, float("inf"), big)
    want = u[:, None] * B[0, :, 3].float()[None] + 1.0
    assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ncols", [8, 64, 65, 300])
def test_lora_infinite_activations_with_positive_adapters(q4k, ncols, dtype):
    """No terms of two signs: an infinite x, A or B makes its sums infinite and none NaN."""
    import torch
    d = make(ncols, ncols, 200, 140, 2, 40, dtype, ids="runs", ragged=False)
    for k in ("A", "B"):
        d[k] = d[k].abs() + 0.5
    d["x"] = d["x"].abs() + 0.5
    hit = torch.zeros(ncols, dtype=torch.bool, device="cuda")
    hit[::3] = True
    d["x"][hit, 77] = float("inf")
    run = lambda: q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], ranks=d["ranks"], scales=d["scales"])  # noqa: E731
    got = run()
    assert (got[hit] == float("inf")).all() and torch.isfinite(got[~hit]).all()
    d["A"][0, 3, 5] = d["B"][1, 7, 9] = float("inf")
    got = run()
    assert (got[hit | (d["ids"] == 0)] == float("inf")).all()
    rest = ~hit & (d["ids"] == 1)
    assert (got[rest][:, 7] == float("inf")).all()
    assert torch.isfinite(got[rest][:, torch.arange(140) != 7]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(300, 8, 256, 1, 64), (300, 8, 256, 1, 128), (70, 100, 33, 1, 200), (300, 8, 384, 1, 512),
                                   (200, 1024, 512, 2, 512), (64, 8, 256, 1, 512)], ids=lambda s: "x".join(map(str, s)))
def test_lora_accuracy_of_terms_of_one_sign(q4k, shape, dtype):
    """Positive x, A and B: sums that are cut off instead of rounded would all err to one side, the more the larger the
    rank. The bound is that of the file's head: sqrt(n) * 2^-24 of the 2-norm, n = K + rank + 1."""
    import torch
    ncols, K, N, slots, rank = shape
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    t = getattr(torch, dtype)
    x, A, B = (torch.rand(s, device="cuda", generator=g) + 0.5 for s in ((ncols, K), (slots, rank, K), (slots, N, rank)))
    d = dict(x=x, A=A.to(t), B=B.to(t), ids=torch.arange(ncols, dtype=torch.int32, device="cuda") % slots)
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"])
    want = reference(d, use_base=False)
    err = torch.linalg.norm(got.double() - want).item() / torch.linalg.norm(want).item()
    assert err <= (K + rank + 1) ** 0.5 * 2.0 ** -24, err * 2.0 ** 24


@pytest.mark.parametrize("dtype", TYPES)
def test_lora_single_products_of_full_mantissas(q4k, dtype):
    """K = rank = 1 and mantissas of ones behind the first eight bits, the worst for products of pieces. Per product,
    in units of 2^-24 of it: what is left out (at most 2 * 2^-25 of a value's binade) 1, the last sum's cut-off (one step, 2^-23) 2,
    the smaller sums' 2^-7 of that; the product with the scale (1) is exact. Two products: 6.1."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    t = getattr(torch, dtype)
    ncols, N = 300, 500
    x, A, B = (1 + 2.0**-7 - torch.randint(1, 9, s, device="cuda", generator=g) * 2.0**-23 for s in ((ncols, 1), (1, 1, 1), (1, N, 1)))
    x[::2] += torch.rand(x[::2].shape, device="cuda", generator=g)
    B[:, ::2] += torch.rand(B[:, ::2].shape, device="cuda", generator=g)
    d = dict(x=x, A=A.to(t), B=B.to(t), ids=torch.zeros(ncols, dtype=torch.int32, device="cuda"))
    want = reference(d, use_base=False)
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"])
    err = ((got.double() - want) / want).abs().max().item()
    assert err <= 6.1 * 2.0 ** -24, err * 2.0 ** 24
