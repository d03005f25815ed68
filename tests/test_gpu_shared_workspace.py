"""One workspace for several kinds of calls in turn: the single-launch GEMV
(gemv_batch_persistent) relies on control words at the start of the workspace that must
come out of every other call as they were."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_lora import make, reference, check_exact
from test_gpu_persistent import MISTRAL, MISTRAL_X, control_words_zero, layer, n_rowgroups

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def step(q4k):
    """A decoder layer for the single-launch path: (run into new outputs, expected outputs)."""
    import torch
    dev = torch.device("cuda")
    _, Wd, xs = layer(q4k, torch, dev, 7, MISTRAL, MISTRAL_X, 1, on_device=True)

    def run(ws):
        out = [torch.full((1, r), float("nan"), device=dev) for r, _ in MISTRAL]
        tasks = q4k.make_tasks(Wd, xs, out)
        assert q4k.batch_persistent_kernel(tasks, 1) == "k_gemv (single launch)"
        q4k.gemv_batch_persistent(tasks, 1, ws)
        return out
    return run, run(q4k.Workspace())


def same(got, want):
    return all(bool((g == w).all()) for g, w in zip(got, want))


def test_adapters_of_many_columns_between_single_launch_calls(q4k, step):
    run, want = step
    ws = q4k.Workspace(1 << 24)  # room for both: it never grows, so it is zeroed once
    assert same(run(ws), want)
    ptr = ws.ptr
    for ncols in (200, 3000):
        d = make(ncols, ncols, 256, 96, 40, 24, "float16")
        got = q4k.lora_add(d["x"], d["A"], d["B"], d["ids"], base=d["base"], ranks=d["ranks"], scales=d["scales"], ws=ws)
        check_exact(got, reference(d))
        assert control_words_zero(ws, n_rowgroups(MISTRAL, 1))
        for _ in range(2):
            assert same(run(ws), want)
    assert ws.ptr == ptr and ws.status() == 0 and np.prod(ws.buf.shape) == 1 << 24


@pytest.mark.parametrize("rows,ncols", [(32, 8), (64, 3), (160, 2), (333, 1)])
def test_smaller_calls_between_single_launch_calls(q4k, step, rows, ncols):
    """Calls of fewer row groups, whose partial sums and activation records follow their own counters."""
    import torch
    run, want = step
    ws = q4k.Workspace(1 << 24)
    assert same(run(ws), want)
    rng = np.random.default_rng(rows)
    W = torch.from_numpy(q4k.gen_q4k_numpy(rng, rows, 14336)).cuda()
    x = torch.from_numpy(rng.standard_normal((ncols, 14336)).astype(np.float32)).cuda()
    alone = q4k.mul_mat_vec_q(W, x, ws=q4k.Workspace())
    y = torch.empty_like(alone)
    tasks = q4k.make_tasks([W], [x], [y])
    for call in (lambda: q4k.mul_mat_vec_q(W, x, out=y, ws=ws), lambda: q4k.gemv_batch(tasks, ncols, ws),
                 lambda: q4k.gemv_batch_persistent(tasks, ncols, ws)):
        y.fill_(float("nan"))
        call()
        assert torch.equal(y, alone)
        assert same(run(ws), want)
    assert ws.status() == 0 and control_words_zero(ws, n_rowgroups(MISTRAL, 1))


def test_counters_have_the_same_room_in_every_workspace(q4k):
    """16384 row groups' counters behind the header, whatever the call."""
    assert q4k.gemv_workspace_bytes(32, 256, 1) >= 256 + 16384 * 4
