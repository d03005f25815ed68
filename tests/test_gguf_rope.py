"""Rotary parameters read from a model file's metadata (GGUFModel.rope): what the file
asks for is given, and what it asks for that cannot be given is refused."""
from __future__ import annotations

import importlib

import numpy as np
import pytest


@pytest.fixture(scope="module")
def loader(q4k):
    return importlib.import_module("q4k_b200.gguf_loader")


@pytest.fixture
def rope(q4k, loader, tmp_path):
    """rope(arch, metadata without the architecture's prefix, ...) of a file with that metadata."""
    def read(arch, meta, extra=None, **kw):
        loader.write_q4k_gguf(tmp_path / "m.gguf", {}, arch=arch, extra_f32=extra or {"t": np.ones(4, np.float32)},
                              metadata={f"{arch}.{k}": v for k, v in meta.items()})
        return loader.GGUFModel(tmp_path / "m.gguf").rope(q4k, device="cpu", **kw)
    return read


def freqs(n_rot, base=10000.0):
    return base ** (-np.arange(n_rot // 2) * 2.0 / n_rot)


def test_rotated_width(rope):
    """The file's count of rotated values, else the length of its keys, else its embedding's share per head."""
    heads = {"embedding_length": 1024, "attention.head_count": 32}
    for meta, want in (({**heads}, 32), ({**heads, "attention.key_length": 128}, 128),
                       ({**heads, "attention.key_length": 128, "rope.dimension_count": 64}, 64),
                       ({"attention.key_length": 80}, 80),
                       ({"embedding_length": 1024, "attention.head_count": [16, 16]}, 64)):
        p = rope("llama", meta)
        assert np.allclose(p["inv_freq"].numpy(), freqs(want), rtol=1e-14) and p["sections"] == (want // 2,)
    for meta in ({}, {"embedding_length": 1024}, {"embedding_length": 1024, "attention.head_count": [16, 8]},
                 {"embedding_length": 1024, "attention.head_count": 0}):
        with pytest.raises(KeyError):
            rope("llama", meta)


def test_scaling(rope):
    """A factor without a type is linear, type none scales nothing, and what is not a factor on the frequencies is refused."""
    d = {"rope.dimension_count": 64, "rope.freq_base": 50000.0}
    for meta, by in (({}, 1.0), ({"rope.scaling.type": "linear", "rope.scaling.factor": 4.0}, 4.0), ({"rope.scaling.factor": 4.0}, 4.0),
                     ({"rope.scaling.type": "none", "rope.scaling.factor": 4.0}, 1.0), ({"rope.scaling.type": "linear"}, 1.0),
                     ({"rope.scaling.factor": 0.0}, 1.0), ({"rope.scale_linear": 2.0}, 2.0), ({"rope.scaling.attn_factor": 1.0}, 1.0),
                     ({"rope.freq_base_swa": 50000.0}, 1.0)):
        assert np.allclose(rope("llama", {**d, **meta})["inv_freq"].numpy(), freqs(64, 50000.0) / by, rtol=1e-14), meta
    for meta in ({"rope.scaling.type": "yarn", "rope.scaling.factor": 4.0}, {"rope.scaling.type": "yarn"},
                 {"rope.scaling.type": "longrope"}, {"rope.scaling.attn_factor": 1.2}, {"rope.freq_base_swa": 10000.0},
                 {"rope.dimension_count_swa": 32}, {"rope.scaling.alpha": 1000.0}):
        with pytest.raises(ValueError):
            rope("llama", {**d, **meta})
    with pytest.raises(ValueError):
        rope("llama", d, extra={"rope_factors_long.weight": np.ones(32, np.float32), "rope_factors_short.weight": np.ones(32, np.float32)})
    f = np.linspace(1, 8, 32, dtype=np.float32)
    p = rope("llama", {**d, "rope.scaling.factor": 2.0}, extra={"rope_freqs.weight": f})
    assert np.allclose(p["inv_freq"].numpy(), freqs(64, 50000.0) / 2 / f.astype(np.float64), rtol=1e-14)


@pytest.mark.parametrize("arch,layout,order", [("llama", "adjacent", "blocks"), ("command-r", "adjacent", None), ("qwen2", "half", None),
                                               ("qwen2vl", "half", "blocks"), ("qwen3vl", "half", "interleaved")])
def test_layout_and_order_of_known_architectures(rope, arch, layout, order):
    one = rope(arch, {"rope.dimension_count": 64})
    assert (one["layout"], one["sections"], one["order"]) == (layout, (32,), "blocks")
    several = {"rope.dimension_count": 64, "rope.dimension_sections": [12, 10, 10, 0]}
    if order is None:
        with pytest.raises(ValueError, match="order"):
            rope(arch, several)
    else:
        p = rope(arch, several)
        assert (p["layout"], p["sections"], p["order"]) == (layout, (12, 10, 10), order)
    p = rope(arch, several, layout="half", order="interleaved")
    assert (p["layout"], p["order"]) == ("half", "interleaved")


def test_unknown_architectures_are_refused_unless_named(rope):
    d = {"rope.dimension_count": 64}
    with pytest.raises(ValueError, match="layout"):
        rope("somethingnew", d)
    assert rope("somethingnew", d, layout="adjacent")["layout"] == "adjacent"
    with pytest.raises(ValueError, match="order"):
        rope("somethingnew", {**d, "rope.dimension_sections": [20, 12]}, layout="half")
    assert rope("somethingnew", {**d, "rope.dimension_sections": [20, 12]}, layout="half", order="blocks")["sections"] == (20, 12)
