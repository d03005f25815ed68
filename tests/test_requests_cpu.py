"""The per-request entries (adapters, rotary positions, logits controls) without a
GPU: bad arguments are refused with a status and a message before a device is
touched, and calls with nothing to do succeed."""
from __future__ import annotations

import ctypes

import pytest

OK, EINVAL, EWORKSPACE = 0, 1, 5
MB = 1 << 20  # fake addresses far apart; nothing is ever read


def lora_task(q4k, **kw):
    t = q4k.LoraTask()
    v = dict(x=1 * MB, base=2 * MB, dst=3 * MB, A=4 * MB, B=5 * MB, ranks=0, scales=0, K=64, nrows=32, stride_col_x=64,
             stride_col_base=32, stride_col_dst=32, stride_a_slot=8 * 64, stride_a_row=64, stride_b_slot=32 * 8,
             stride_b_row=8, slots=4, rank=8, type=1)
    v.update(kw)
    for k, val in v.items():
        setattr(t, k, val)
    return t


def lora(q4k, tasks, ncols=4, ids=6 * MB, ws=None, wsb=0):
    arr = (q4k.LoraTask * max(1, len(tasks)))(*tasks)
    return q4k.lib().q4k_lora_batch(arr, len(tasks), ncols, ids, ws, wsb, None)


@pytest.mark.parametrize("kw", [
    dict(K=-1), dict(nrows=-1), dict(K=1 << 31), dict(slots=-1), dict(slots=1025), dict(rank=-1), dict(rank=513),
    dict(type=2), dict(dst=0), dict(x=0), dict(A=0), dict(B=0), dict(dst=3 * MB + 2), dict(x=MB + 1), dict(A=4 * MB + 1),
    dict(B=5 * MB + 1), dict(stride_col_x=63), dict(stride_col_x=-64), dict(stride_col_base=31), dict(stride_col_dst=31),
    dict(stride_col_dst=0), dict(stride_a_row=63), dict(stride_b_row=7), dict(stride_a_slot=-1), dict(ranks=3), dict(scales=2),
    dict(base=3 * MB + 4), dict(base=3 * MB, stride_col_base=40), dict(dst=1 * MB), dict(dst=1 * MB + 256),
    dict(stride_col_x=1 << 41), dict(stride_b_slot=-8),
])
def test_lora_refuses(q4k, kw):
    assert lora(q4k, [lora_task(q4k, **kw)]) == EINVAL
    assert len(q4k.lib().q4k_last_error()) > 0


def test_lora_refuses_between_tasks(q4k):
    a = lora_task(q4k)
    assert lora(q4k, [a, lora_task(q4k)]) == EINVAL  # the same dst twice
    assert lora(q4k, [a, lora_task(q4k, dst=7 * MB, base=0, x=3 * MB)]) == EINVAL  # reads what the other writes
    assert lora(q4k, [a, lora_task(q4k, dst=7 * MB, base=3 * MB)]) == EINVAL
    assert lora(q4k, [a, lora_task(q4k, dst=7 * MB, base=0, type=30)]) == EINVAL  # two types
    assert lora(q4k, [a] * 17) == EINVAL
    assert lora(q4k, [a], ncols=-1) == EINVAL
    assert lora(q4k, [a], ids=0) == EINVAL
    assert lora(q4k, [a], ids=6 * MB + 2) == EINVAL


def test_lora_nothing_to_do(q4k):
    assert lora(q4k, []) == OK
    assert lora(q4k, [lora_task(q4k)], ncols=0) == OK
    assert lora(q4k, [lora_task(q4k, nrows=0)]) == OK


def test_lora_workspace_refused(q4k):
    t = (q4k.LoraTask * 1)(lora_task(q4k, K=4096, stride_col_x=4096, stride_a_row=4096, stride_a_slot=8 * 4096,
                                     x=64 * MB))
    need = q4k.lib().q4k_lora_workspace_bytes(t, 1, 1000)
    assert need > 0
    for ws, wsb in ((None, need), (256 * MB, need - 1), (256 * MB + 16, need)):
        assert q4k.lib().q4k_lora_batch(t, 1, 1000, 6 * MB, ws, wsb, None) == EWORKSPACE
    bad = (q4k.LoraTask * 1)(lora_task(q4k, rank=-1))
    assert q4k.lib().q4k_lora_workspace_bytes(bad, 1, 1000) == 0


def rope(q4k, ncols=4, dim=64, n_rot=64, pos=8 * MB, sp=4, inv=9 * MB, sections=(16, 8, 8), order=0, layout=0, dst_type=0,
         n=1, tensors=None, **kw):
    v = dict(x=1 * MB, dst=2 * MB, stride_col_x=8 * 64, stride_head_x=64, stride_col_dst=8 * 64, stride_head_dst=64,
             heads=8)
    v.update(kw)
    t = q4k.RopeTensor(**v)
    arr = (q4k.RopeTensor * max(1, n))(*(tensors or [t] * n))
    s = (ctypes.c_int * max(1, len(sections)))(*sections) if sections is not None else None
    return q4k.lib().q4k_rope_multi(arr, n, ncols, dim, n_rot, pos, sp, inv, s, len(sections or (1,)), order, layout,
                                    1.0, dst_type, None)


@pytest.mark.parametrize("kw", [
    dict(ncols=-1), dict(dim=0), dict(dim=1025), dict(n_rot=63), dict(n_rot=66), dict(n_rot=-2), dict(sections=()),
    dict(sections=(1, 1, 1, 1, 1)), dict(sections=(0, 0)), dict(sections=(-1, 33)), dict(sections=None), dict(order=2),
    dict(layout=2), dict(dst_type=2), dict(pos=0), dict(pos=8 * MB + 2), dict(inv=0), dict(inv=9 * MB + 4), dict(sp=3),
    dict(x=0), dict(dst=0), dict(x=MB + 2), dict(dst=2 * MB + 2), dict(heads=-1), dict(stride_head_dst=63),
    dict(stride_col_dst=8 * 64 - 1), dict(stride_col_x=-1), dict(n=5), dict(n=-1),
    dict(dst=1 * MB + 256), dict(dst=1 * MB, dst_type=1), dict(dst=1 * MB, stride_col_dst=8 * 64 + 64),
])
def test_rope_refuses(q4k, kw):
    assert rope(q4k, **kw) == EINVAL
    assert len(q4k.lib().q4k_last_error()) > 0


def test_rope_refuses_between_tensors(q4k):
    def t(x, dst):
        return q4k.RopeTensor(x=x, dst=dst, stride_col_x=512, stride_head_x=64, stride_col_dst=512, stride_head_dst=64,
                              heads=8)
    assert rope(q4k, n=2, tensors=[t(MB, 2 * MB), t(3 * MB, 2 * MB)]) == EINVAL
    assert rope(q4k, n=2, tensors=[t(MB, 2 * MB), t(2 * MB, 3 * MB)]) == EINVAL
    assert rope(q4k, ncols=0) == OK
    assert rope(q4k, n=0) == OK
    assert rope(q4k, heads=0) == OK


def logits(q4k, ncols=4, **kw):
    v = dict(logits=1 * MB, dst=2 * MB, nvocab=100, stride_col=100, stride_col_dst=100, history=3 * MB,
             history_len=4 * MB, penalties=5 * MB, max_history=16, stride_history=16, bias_tokens=6 * MB,
             bias_values=7 * MB, bias_offsets=8 * MB, n_bias=10, mask=9 * MB, mask_rows=10 * MB, stride_mask=4, n_masks=2,
             token=11 * MB, lse=12 * MB)
    v.update(kw)
    return q4k.lib().q4k_logits_process(ctypes.byref(q4k.LogitsArgs(**v)), ncols, None)


@pytest.mark.parametrize("kw", [
    dict(ncols=-1), dict(nvocab=-1), dict(nvocab=1 << 31), dict(max_history=-1), dict(n_bias=-1), dict(n_masks=-1),
    dict(logits=0), dict(dst=0), dict(logits=MB + 2), dict(dst=2 * MB + 1), dict(stride_col=99), dict(stride_col_dst=99),
    dict(stride_col_dst=0), dict(history=0), dict(penalties=0), dict(stride_history=15), dict(bias_tokens=0),
    dict(bias_values=0), dict(bias_offsets=0), dict(mask=0), dict(stride_mask=3), dict(history=3 * MB + 1),
    dict(token=11 * MB + 2), dict(lse=12 * MB + 2), dict(mask=9 * MB + 2), dict(dst=1 * MB + 4),
    dict(dst=1 * MB, stride_col_dst=200),
])
def test_logits_refuses(q4k, kw):
    assert logits(q4k, **kw) == EINVAL
    assert len(q4k.lib().q4k_last_error()) > 0


def test_logits_nothing_to_do(q4k):
    assert logits(q4k, ncols=0) == OK
    assert q4k.lib().q4k_logits_process(None, 1, None) == EINVAL


def test_python_wrappers_refuse_cpu_tensors(q4k):
    import torch
    x = torch.zeros(2, 8)
    for call in (lambda: q4k.lora_add(x, torch.zeros(1, 2, 8), torch.zeros(1, 4, 2), torch.zeros(2, dtype=torch.int32)),
                 lambda: q4k.rope_multi(torch.zeros(2, 1, 8), torch.zeros(1, 2, dtype=torch.int32),
                                        torch.zeros(4, dtype=torch.float64), (4,)),
                 lambda: q4k.logits_process(x)):
        with pytest.raises(q4k.Q4KError) as e:
            call()
        assert e.value.status == EINVAL


def test_structures_match_the_header(q4k):
    """The ctypes structures are as large as the native front-end's C structs (one task's bytes)."""
    import torch
    assert q4k._native().lora_pack([]) == b""
    assert ctypes.sizeof(q4k.LoraTask) == 7 * 8 + 9 * 8 + 4 * 4
    assert ctypes.sizeof(q4k.RopeTensor) == 2 * 8 + 4 * 8 + 8
    assert ctypes.sizeof(q4k.LogitsArgs) == 20 * 8
    with pytest.raises(q4k.Q4KError):
        q4k.lora_batch([dict(x=torch.zeros(1, 8))], torch.zeros(1, dtype=torch.int32))
    assert q4k.lora_batch([], torch.zeros(1, dtype=torch.int32)) == []


def test_lora_batch_takes_no_other_array(q4k):
    """Arrays of GEMV tasks, and adapter tasks whose number of columns nobody checked, are refused."""
    import torch
    ids = torch.zeros(1, dtype=torch.int32)
    for arr in ((q4k.Task * 2)(), (q4k.TaskEx * 1)(), (ctypes.c_char * 144)(), (q4k.LoraTask * 1)()):
        with pytest.raises(q4k.Q4KError, match="make_lora_tasks"):
            q4k.lora_batch(arr, ids)
    with pytest.raises(q4k.Q4KError, match="bytes"):  # not a whole number of tasks
        q4k._native().lora_run(bytes(ctypes.sizeof(q4k.LoraTask) + 8), ids, None, None, 1, 0)
    assert q4k.lora_batch(q4k.make_lora_tasks([]), ids) is None
