"""Adapter files into slots (gguf_loader.load_adapters): values come through as the files
hold them."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

NAMES = ["blk.0.attn_q.weight", "blk.0.attn_k.weight"]


@pytest.fixture(scope="module")
def loader(q4k):
    return importlib.import_module("q4k_b200.gguf_loader")


def write(loader, path, kind, seed, names=NAMES, values=()):
    """An adapter file of that element type; returns name -> (A, B) as fp32 arrays of the values it holds."""
    import gguf
    import torch
    rng = np.random.default_rng(seed)
    held, mats = {}, {}
    for name in names:
        pair = [rng.standard_normal(s).astype(np.float32) for s in ((4, 32), (24, 4))]
        for i, v in enumerate(values):
            pair[i % 2].flat[i] = v
        if kind != "float32":
            pair = [torch.from_numpy(p).to(getattr(torch, kind)).float().numpy() for p in pair]
        held[name] = pair
        mats[name] = [p.astype(np.float16) for p in pair] if kind == "float16" else pair
    if kind != "bfloat16":
        loader.write_adapter_gguf(path, mats, alpha=4.0)
        return held
    w = gguf.GGUFWriter(str(path), "llama")
    w.add_string("adapter.type", "lora")
    w.add_float32("adapter.lora.alpha", 4.0)
    for name, pair in mats.items():
        for end, a in zip(("lora_a", "lora_b"), pair):
            w.add_tensor(f"{name}.{end}", gguf.quants.quantize(a, gguf.GGMLQuantizationType.BF16),
                         raw_dtype=gguf.GGMLQuantizationType.BF16)
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()
    return held


@pytest.mark.parametrize("kinds,want", [(("float16",), "float16"), (("bfloat16",), "bfloat16"), (("float32",), "float32"),
                                        (("float16", "bfloat16"), "float32"), (("float16", "float32"), "float32")])
def test_adapters_keep_their_files_type_and_values(loader, tmp_path, kinds, want):
    import torch
    beyond = {"float32": (7e4, 1e-8, -3e38, 1 / 3), "bfloat16": (7e4, 1e-8, -3e38, 1.0), "float16": (65504.0, 6e-8, 1.0, -2.0)}
    held = [write(loader, tmp_path / f"{i}.gguf", k, i, values=beyond[k]) for i, k in enumerate(kinds)]
    got = loader.load_adapters([tmp_path / f"{i}.gguf" for i in range(len(kinds))], NAMES, device="cpu")
    for name in NAMES:
        for s, h in enumerate(held):
            t = got[name]
            assert t["A"].dtype == t["B"].dtype == getattr(torch, want)
            assert np.array_equal(t["A"][s, :4].float().numpy(), h[name][0]) and np.array_equal(t["B"][s, :, :4].float().numpy(), h[name][1])


def test_adapters_of_one_call_have_one_type(loader, tmp_path):
    """A matrix only fp16 files adapt, beside one that an fp32 file adapts: lora_batch takes one type per call."""
    import torch
    write(loader, tmp_path / "a.gguf", "float16", 1)
    write(loader, tmp_path / "b.gguf", "float32", 2, names=NAMES[1:])
    got = loader.load_adapters([tmp_path / "a.gguf", tmp_path / "b.gguf"], NAMES, device="cpu")
    assert {t["A"].dtype for t in got.values()} == {torch.float32}
    got = loader.load_adapters([tmp_path / "a.gguf", tmp_path / "b.gguf"], NAMES[:1], device="cpu")
    assert got[NAMES[0]]["A"].dtype == torch.float16


def test_a_type_that_cannot_hold_the_values_is_refused(loader, tmp_path):
    import torch
    held = write(loader, tmp_path / "a.gguf", "float32", 1, values=(7e4,))
    with pytest.raises(OverflowError):
        loader.load_adapters([tmp_path / "a.gguf"], NAMES, device="cpu", dtype=torch.float16)
    got = loader.load_adapters([tmp_path / "a.gguf"], NAMES, device="cpu", dtype=torch.bfloat16)
    want = torch.from_numpy(held[NAMES[0]][0]).bfloat16()
    assert torch.equal(got[NAMES[0]]["A"][0, :4], want)
    write(loader, tmp_path / "b.gguf", "float32", 1, values=(np.inf,))  # the file's own infinity stays
    got = loader.load_adapters([tmp_path / "b.gguf"], NAMES, device="cpu", dtype=torch.float16)
    assert torch.isinf(got[NAMES[0]]["A"][0, 0, 0])
