"""GGUF loading: Q4_K weight tensors of an on-disk model into device memory,
in the layout the GEMV entries take (one row per 256-weight super-block run,
144 bytes per super-block, rows contiguous).

The reference runs llama.cpp on a Q4_K GGUF checkpoint
(`llama-cli ... mistral-7b-v0.3-q4.gguf`); this is the path from such a file
to `q4k_gemv_batch` tasks.  Parsing uses the `gguf` package (gguf-py, the
format's reference reader); the file is memory-mapped and each tensor is
copied to the device once.  GGUF stores a matrix as ne = [K, rows] with rows
contiguous: exactly the Q4_K row layout, so no repacking is needed.

Names follow llama.cpp's tensor naming (`blk.{i}.attn_q.weight`, ...).
Adapter files (`load_adapters`) and the rotary parameters (`GGUFModel.rope`)
come the same way, in the form q4k.lora_batch and q4k.rope_multi take.
"""
from __future__ import annotations

from dataclasses import dataclass
from pathlib import Path

import numpy as np

QK_K = 256
BLOCK_BYTES = 144

# llama-style decoder layer matrices, in the order of a layer's launch group
# (activation group: attn = attn_norm(x), o = attention output, ffn =
# ffn_norm(h), down = glu(gate, up)).
LLAMA_LAYER = (("q", "attn_q", "attn"), ("k", "attn_k", "attn"), ("v", "attn_v", "attn"),
               ("o", "attn_output", "o"), ("gate", "ffn_gate", "ffn"), ("up", "ffn_up", "ffn"),
               ("down", "ffn_down", "down"))

# How an architecture's files store the rotated pairs of q and k (neighbours, or
# halves of the rotated width), and how it deals its pairs out to several axes.
ROPE_LAYOUTS = {
    **dict.fromkeys(("llama", "baichuan", "command-r", "cohere2", "deepseek", "granite", "granitemoe", "internlm2",
                     "minicpm", "olmo", "smollm3", "xverse"), "adjacent"),
    **dict.fromkeys(("exaone", "falcon", "gemma", "gemma2", "gptneox", "nemotron", "olmo2", "olmoe", "orion", "phi2", "phi3",
                     "qwen2", "qwen2moe", "qwen2vl", "qwen3", "qwen3moe", "qwen3vl", "qwen3vlmoe", "stablelm",
                     "starcoder2"), "half"),
}
ROPE_ORDERS = {"llama": "blocks", "qwen2vl": "blocks", "qwen3vl": "interleaved", "qwen3vlmoe": "interleaved"}


@dataclass
class Q4KTensor:
    """One Q4_K matrix: `data` is (rows, K/256*144) uint8 (numpy memmap view or device tensor)."""
    name: str
    rows: int
    K: int
    data: object


class GGUFModel:
    """A GGUF file opened for reading (memory-mapped)."""

    def __init__(self, path: str | Path):
        import gguf
        self._gguf = gguf
        self.path = Path(path)
        self.reader = gguf.GGUFReader(str(self.path), "r")
        self.tensors = {t.name: t for t in self.reader.tensors}

    # ---- metadata ---------------------------------------------------------
    def field(self, key: str):
        """A scalar or string metadata value (None when absent)."""
        f = self.reader.fields.get(key)
        if f is None or not f.types:
            return None
        part = f.parts[f.data[0]]
        if f.types[0] == self._gguf.GGUFValueType.STRING:
            return bytes(part).decode("utf-8")
        return part.tolist()[0] if len(part) == 1 else part.tolist()

    @property
    def arch(self) -> str | None:
        return self.field("general.architecture")

    def n_layers(self) -> int:
        n = self.field(f"{self.arch}.block_count") if self.arch else None
        if n is not None:
            return int(n)
        idx = {int(name.split(".")[1]) for name in self.tensors if name.startswith("blk.")}
        return max(idx) + 1 if idx else 0

    def array(self, key: str) -> list | None:
        """An array metadata value as a list (None when absent)."""
        f = self.reader.fields.get(key)
        if f is None:
            return None
        return [v for i in f.data for v in np.asarray(f.parts[i]).tolist()]

    def rope(self, q4k, layout: str | None = None, order: str | None = None, device="cuda") -> dict:
        """Keyword arguments for q4k.rope_multi (inv_freq, sections, layout, order) from the
        metadata `<arch>.rope.*` and the `rope_freqs.weight` factors.  Sections are the
        M-RoPE `dimension_sections` without trailing zeros (one axis where there are none).
        Without a `dimension_count` heads turn whole: `attention.key_length` values, else
        the embedding's share of a head.  A `scaling.factor` divides the frequencies unless
        the file's `scaling.type` is none; files that ask for another scaling (yarn,
        longrope) or for a second set of frequencies are refused.  layout, and order where
        there are several axes, have to be given for an architecture that ROPE_LAYOUTS and
        ROPE_ORDERS do not know."""
        a = self.arch
        n_rot = self.field(f"{a}.rope.dimension_count")
        if n_rot is None:  # whole heads
            n_rot = self.field(f"{a}.attention.key_length")
        if n_rot is None:
            heads = set(self.array(f"{a}.attention.head_count") or [])  # one number, or one per layer
            width = self.field(f"{a}.embedding_length")
            if len(heads) != 1 or 0 in heads or not width:
                raise KeyError(f"{self.path}: no {a}.rope.dimension_count, nor the width of a head")
            n_rot = int(width) // int(heads.pop())
        base = self.field(f"{a}.rope.freq_base") or 10000.0
        kind = self.field(f"{a}.rope.scaling.type") or "linear"
        if kind not in ("linear", "none"):
            raise ValueError(f"{self.path}: rotary scaling {kind!r} (only linear scaling and none)")
        # other frequencies for long contexts or for windowed layers, or a factor on the turned values
        for key, same in (("rope.scaling.attn_factor", 1.0), ("rope.scaling.alpha", 0.0), ("rope.freq_base_swa", base),
                          ("rope.dimension_count_swa", n_rot)):
            v = self.field(f"{a}.{key}")
            if v is not None and v != same:
                raise ValueError(f"{self.path}: {a}.{key} = {v} is not supported")
        if "rope_factors_long.weight" in self.tensors or "rope_factors_short.weight" in self.tensors:
            raise ValueError(f"{self.path}: rotary factors by context length are not supported")
        factor = self.field(f"{a}.rope.scaling.factor") or self.field(f"{a}.rope.scale_linear")
        scale = 1.0 / factor if kind == "linear" and factor else 1.0
        t = self.tensors.get("rope_freqs.weight")
        sections = [int(v) for v in self.array(f"{a}.rope.dimension_sections") or []]
        while sections and sections[-1] == 0:
            sections.pop()
        layout = layout or ROPE_LAYOUTS.get(a)
        order = order or (ROPE_ORDERS.get(a) if len(sections) > 1 else "blocks")
        if layout is None or order is None:
            raise ValueError(f"{self.path}: architecture {a!r}: give the rotary {'order' if layout else 'layout'}")
        return dict(inv_freq=q4k.rope_inv_freq(int(n_rot), base, scale, None if t is None else np.array(t.data), device=device),
                    sections=tuple(sections) or (int(n_rot) // 2,),
                    layout=layout, order=order)

    # ---- tensors ----------------------------------------------------------
    def q4k(self, name: str) -> Q4KTensor:
        """Host view of one Q4_K matrix; raises for another type or a shape that is not rows x K."""
        t = self.tensors.get(name)
        if t is None:
            raise KeyError(f"{self.path}: no tensor {name!r}")
        if t.tensor_type != self._gguf.GGMLQuantizationType.Q4_K:
            raise TypeError(f"{name}: type {t.tensor_type.name}, not Q4_K")
        dims = [int(d) for d in t.shape]  # ggml order: ne0 = K, ne1 = rows, higher dims 1
        if len(dims) < 2 or any(d != 1 for d in dims[2:]):
            raise ValueError(f"{name}: shape {dims} is not a matrix")
        K, rows = dims[0], dims[1]
        if K % QK_K:
            raise ValueError(f"{name}: K={K} is not a multiple of {QK_K}")
        data = np.asarray(t.data).reshape(rows, K // QK_K * BLOCK_BYTES)
        return Q4KTensor(name, rows, K, data)

    def q4k_names(self) -> list[str]:
        return [n for n, t in self.tensors.items() if t.tensor_type == self._gguf.GGMLQuantizationType.Q4_K]

    def to_device(self, name: str, device="cuda", stream=None) -> Q4KTensor:
        """Copy one Q4_K matrix to the device (16-byte aligned, rows contiguous)."""
        import torch
        h = self.q4k(name)
        src = torch.from_numpy(np.ascontiguousarray(h.data))  # the memmap is read-only: one host copy
        dst = torch.empty(src.shape, dtype=torch.uint8, device=device)
        if stream is None:
            dst.copy_(src)
        else:
            with torch.cuda.stream(stream):
                dst.copy_(src, non_blocking=False)
        return Q4KTensor(name, h.rows, h.K, dst)

    def layer(self, i: int, device="cuda") -> dict[str, Q4KTensor]:
        """The seven Q4_K matrices of decoder layer i (llama naming), on the device."""
        out = {}
        for key, stem, _ in LLAMA_LAYER:
            out[key] = self.to_device(f"blk.{i}.{stem}.weight", device)
        return out


def layer_tasks(q4k, layer: dict[str, Q4KTensor], xs: dict, outs: dict, fuse_ffn: bool = False):
    """Task array for one decoder layer: xs maps activation group -> (ncols, K)
    fp32 device tensor, outs maps matrix key -> (ncols, rows) output.  With
    fuse_ffn the gate and up matrices become one task with the SwiGLU
    epilogue (output in outs["up"]), as llama.cpp's fused Q4_K FFN call."""
    groups = {key: grp for key, _, grp in LLAMA_LAYER}
    if not fuse_ffn:
        keys = [key for key, _, _ in LLAMA_LAYER]
        return q4k.make_tasks([layer[k].data for k in keys], [xs[groups[k]] for k in keys],
                              [outs[k] for k in keys])
    items = []
    for key, _, grp in LLAMA_LAYER:
        if key == "gate":
            continue
        it = dict(W=layer[key].data, x=xs[grp], out=outs[key])
        if key == "up":
            it.update(W_gate=layer["gate"].data, glu="swiglu")
        items.append(it)
    return q4k.make_tasks_ex(items)


# ---- low-rank adapters -----------------------------------------------------------
def load_adapters(paths, names, device="cuda", dtype=None, strengths=None) -> dict[str, dict]:
    """Adapter files (llama.cpp's `adapter.type = lora`: `<tensor>.lora_a` with ne = [K, rank],
    `<tensor>.lora_b` with ne = [rank, rows]) stacked into slots, slot s = paths[s], for the
    matrices `names` (e.g. "blk.0.attn_q.weight"): name -> dict(A, B, ranks, scales) as
    q4k.lora_batch takes them.  dtype: by default the files' own where all of these
    matrices are fp16 or all bf16, else fp32; values that are finite in the file and not in
    a given dtype are refused.  The scale of a slot is
    strengths[s] * alpha / rank (strengths[s] where the file's alpha is 0 or missing); a
    matrix that a file does not adapt has rank 0 in its slot; ranks are padded to a
    multiple of 8 so that rows stay 16-byte aligned.  Matrices that no file adapts are
    left out."""
    import gguf
    import torch
    names = list(names)
    files = []
    for path in paths:
        m = GGUFModel(path)
        if m.field("adapter.type") not in (None, "lora"):
            raise TypeError(f"{path}: adapter.type {m.field('adapter.type')!r}, not lora")
        files.append((m, float(m.field("adapter.lora.alpha") or 0.0)))
    strengths = [1.0] * len(files) if strengths is None else list(strengths)
    if len(strengths) != len(files):
        raise ValueError(f"{len(strengths)} strengths for {len(files)} adapters")

    def matrix(t) -> np.ndarray:
        if t.tensor_type in (gguf.GGMLQuantizationType.F32, gguf.GGMLQuantizationType.F16):
            a = np.asarray(t.data).astype(np.float32)
        else:  # bf16 and quantized adapters
            a = gguf.quants.dequantize(np.asarray(t.data), t.tensor_type)
        return np.ascontiguousarray(a.reshape([int(d) for d in t.shape][::-1][-2:]))

    if dtype is None:  # one for all: a launch takes adapters of one type
        Q = gguf.GGMLQuantizationType
        kinds = {m.tensors[key].tensor_type for m, _ in files for name in names
                 for key in (name + ".lora_a", name + ".lora_b") if key in m.tensors}
        dtype = torch.float16 if kinds == {Q.F16} else torch.bfloat16 if kinds == {Q.BF16} else torch.float32

    def converted(a: np.ndarray, path, name: str):
        t = torch.from_numpy(a)
        c = t.to(dtype)
        if not torch.equal(torch.isfinite(c), torch.isfinite(t)):
            raise OverflowError(f"{path}: {name}: values beyond {dtype}")
        return c

    out = {}
    for name in names:
        pairs = []
        for m, _ in files:
            a, b = m.tensors.get(name + ".lora_a"), m.tensors.get(name + ".lora_b")
            if (a is None) != (b is None):
                raise KeyError(f"{m.path}: {name} has only one of lora_a and lora_b")
            pairs.append(None if a is None else (matrix(a), matrix(b)))
        some = [p for p in pairs if p is not None]
        if not some:
            continue
        K, rows = some[0][0].shape[1], some[0][1].shape[0]
        for (m, _), p in zip(files, pairs):
            if p is not None and (p[0].shape[1] != K or p[1].shape != (rows, p[0].shape[0])):
                raise ValueError(f"{m.path}: {name}: shapes {p[0].shape} and {p[1].shape}")
        rank = (max(p[0].shape[0] for p in some) + 7) // 8 * 8
        A, B = torch.zeros((len(files), rank, K), dtype=dtype), torch.zeros((len(files), rows, rank), dtype=dtype)
        ranks, scales = torch.zeros(len(files), dtype=torch.int32), torch.zeros(len(files), dtype=torch.float32)
        for s, p in enumerate(pairs):
            if p is None:
                continue
            r = p[0].shape[0]
            A[s, :r], B[s, :, :r] = (converted(a, files[s][0].path, name) for a in p)
            ranks[s] = r
            scales[s] = strengths[s] * (files[s][1] / r if files[s][1] and r else 1.0)
        out[name] = dict(A=A.to(device), B=B.to(device), ranks=ranks.to(device), scales=scales.to(device))
    return out


def layer_adapter_items(adapters: dict[str, dict], i: int, xs: dict, outs: dict) -> list[dict]:
    """Items for q4k.lora_batch that add the adapters of decoder layer i to the outputs of its
    layer_tasks launch, in place (xs, outs: as for layer_tasks, unfused)."""
    items = []
    for key, stem, grp in LLAMA_LAYER:
        ad = adapters.get(f"blk.{i}.{stem}.weight")
        if ad is not None and key in outs:
            items.append(dict(x=xs[grp], base=outs[key], out=outs[key], **ad))
    return items


def write_adapter_gguf(path: str | Path, mats: dict[str, tuple[np.ndarray, np.ndarray]], alpha: float,
                       arch: str = "llama") -> None:
    """Write an adapter file: name -> (A (rank, K), B (rows, rank)) in fp16 or fp32."""
    import gguf
    w = gguf.GGUFWriter(str(path), arch)
    w.add_string("general.type", "adapter")
    w.add_string("adapter.type", "lora")
    w.add_float32("adapter.lora.alpha", float(alpha))
    for name, (a, b) in mats.items():
        w.add_tensor(name + ".lora_a", np.ascontiguousarray(a))
        w.add_tensor(name + ".lora_b", np.ascontiguousarray(b))
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()


def write_q4k_gguf(path: str | Path, tensors: dict[str, np.ndarray], arch: str = "llama",
                   extra_f32: dict[str, np.ndarray] | None = None, n_layers: int | None = None,
                   metadata: dict | None = None) -> None:
    """Write a GGUF file holding Q4_K matrices given as (rows, K/256*144) uint8
    arrays (and optional fp32 tensors, and metadata of whole numbers, fp32,
    strings and lists of whole numbers): for tests and for staging synthetic
    weights in the on-disk format."""
    import gguf
    w = gguf.GGUFWriter(str(path), arch)
    for key, v in (metadata or {}).items():
        if isinstance(v, (list, tuple)):
            w.add_array(key, list(v))
        else:
            {int: w.add_uint32, float: w.add_float32, str: w.add_string}[type(v)](key, v)
    if n_layers is not None:
        w.add_block_count(n_layers)
    for name, a in tensors.items():
        a = np.ascontiguousarray(a, dtype=np.uint8)
        if a.ndim != 2 or a.shape[1] % BLOCK_BYTES:
            raise ValueError(f"{name}: expected (rows, K/256*144) uint8, got {a.shape}")
        w.add_tensor(name, a, raw_dtype=gguf.GGMLQuantizationType.Q4_K)
    for name, a in (extra_f32 or {}).items():
        w.add_tensor(name, np.ascontiguousarray(a, dtype=np.float32))
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()
