"""The per-request entries on columns, heads, slots and rows that lie more than 2^31 values apart, in buffers that
are mostly never touched."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_logits import check as check_logits
from test_gpu_logits import make as make_logits
from test_gpu_lora import check_exact, make, reference
from test_gpu_rope_multi import check as check_rope

pytestmark = pytest.mark.gpu

FAR = (1 << 30) + 64  # two steps pass 2^31


@pytest.fixture(autouse=True)
def give_back():
    yield
    import torch
    torch.cuda.empty_cache()


def far(shape, strides, dtype, off=0):
    """A view with these strides of a buffer just as long as it needs."""
    import torch
    n = off + sum((s - 1) * st for s, st in zip(shape, strides)) + 1
    return torch.as_strided(torch.empty(n, dtype=dtype, device="cuda"), shape, strides, off)


@pytest.mark.parametrize("extra", [0, 1])
def test_logits_far_apart(q4k, extra):
    import torch
    d = make_logits(3, 3, 5000, hist=20, bias=10, masks=2)
    t = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in d.items()}
    rows = far((3, 5000), (FAR + extra, 1), torch.float32)
    rows.copy_(t.pop("logits"))
    check_logits(q4k.logits_process(rows, **t, out=rows, pick=True), d)


@pytest.mark.parametrize("dim", [64, 62])
@pytest.mark.parametrize("head_major", [False, True])
def test_rope_far_apart(q4k, dim, head_major):
    import torch
    rng = np.random.default_rng(dim)
    x = rng.standard_normal((3, 3, dim)).astype(np.float32)
    pos = rng.integers(0, 4000, (2, 3)).astype(np.int32)
    inv = q4k.rope_inv_freq(dim, 1e4)
    strides = (dim, FAR, 1) if head_major else (FAR, dim, 1)
    view = far((3, 3, dim), strides, torch.float32)
    view.copy_(torch.from_numpy(x))
    q4k.rope_multi(view, torch.from_numpy(pos).cuda(), inv, (10, dim // 2 - 10), out=view)
    check_rope(view, x, pos, inv.cpu().numpy(), (10, dim // 2 - 10))


@pytest.mark.parametrize("ncols", [3, 70])
@pytest.mark.parametrize("what", ["columns", "slots", "rows"])
def test_lora_far_apart(q4k, ncols, what):
    import torch
    K, N, slots, rank = 96, 40, 3, 16
    d = make(ncols, ncols, K, N, slots, rank, "float16", ids="runs")
    want = reference(d)
    step = FAR * 2 // (ncols - 1) // 8 * 8 + 64
    if what == "columns":
        for k, n in (("x", K), ("base", N)):
            view = far((ncols, n), (step, 1), torch.float32)
            view.copy_(d[k])
            d[k] = view
    elif what == "slots":
        for k, inner in (("A", (K, 1)), ("B", (rank, 1))):
            view = far(tuple(d[k].shape), (FAR, *inner), torch.float16)
            view.copy_(d[k])
            d[k] = view
    else:  # the last rows of A and B start behind 2^31 values
        for k, rows in (("A", rank), ("B", N)):
            st = ((1 << 31) // (rows - 1) + 8) // 8 * 8
            view = far(tuple(d[k].shape), (st * rows, st, 1), torch.float16)
            view.copy_(d[k])
            d[k] = view
    got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"],
                       out=d["base"] if what == "columns" else None)
    check_exact(got, want)
