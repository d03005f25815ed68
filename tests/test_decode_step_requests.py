"""A decode step of a batch of requests, as the pieces are used together: a GGUF
checkpoint's layer runs its projections in one batch launch, every request's adapter is
added to them, queries and keys are turned to each request's position, and behind the
output head every request's penalties, biases and mask are applied and its token picked;
eagerly and as one captured graph over changing requests, against 64-bit references."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from test_gpu_logits import reference as logits_reference
from test_gpu_rope_multi import reference as rope_reference

SHAPES = {"attn_q": (512, 512), "attn_k": (128, 512), "attn_v": (128, 512), "attn_output": (512, 512),
          "ffn_gate": (768, 512), "ffn_up": (768, 512), "ffn_down": (512, 768)}
HEAD_DIM = 64
VOCAB = 4000


@pytest.fixture(scope="module")
def loader(q4k):
    return importlib.import_module("q4k_b200.gguf_loader")


@pytest.fixture(scope="module")
def files(q4k, loader, tmp_path_factory):
    rng = np.random.default_rng(11)
    d = tmp_path_factory.mktemp("requests")
    mats = {f"blk.0.{s}.weight": q4k.gen_q4k_numpy(rng, rows, K) for s, (rows, K) in SHAPES.items()}
    mats["output.weight"] = q4k.gen_q4k_numpy(rng, VOCAB, 512)
    loader.write_q4k_gguf(d / "model.gguf", mats, n_layers=1, extra_f32={"rope_freqs.weight": np.linspace(1, 4, 32, dtype=np.float32)},
                          metadata={"llama.rope.dimension_count": HEAD_DIM, "llama.rope.freq_base": 50000.0,
                                    "llama.rope.dimension_sections": [12, 10, 10, 0]})
    adapters = []
    for s, (rank, stems) in enumerate([(8, ("attn_q", "attn_v")), (5, ("attn_q", "attn_k", "ffn_down")), (16, tuple(SHAPES))]):
        a = {f"blk.0.{stem}.weight": (rng.standard_normal((rank, SHAPES[stem][1])).astype(np.float16) / 16,
                                      rng.standard_normal((SHAPES[stem][0], rank)).astype(np.float16)) for stem in stems}
        loader.write_adapter_gguf(d / f"adapter{s}.gguf", a, alpha=0.0 if s == 1 else 16.0)
        adapters.append((rank, a))
    return d, mats, adapters


def load(loader, files, device="cuda"):
    names = [f"blk.0.{s}.weight" for s in SHAPES]
    return loader.load_adapters([files[0] / f"adapter{s}.gguf" for s in range(3)], names, device=device, strengths=[1.0, 0.5, 1.0])


def test_adapter_files_become_slots(q4k, loader, files):
    got = load(loader, files, device="cpu")
    for stem, (rows, K) in SHAPES.items():
        t = got[f"blk.0.{stem}.weight"]
        rank = t["A"].shape[1]
        assert rank % 8 == 0 and t["A"].shape == (3, rank, K) and t["B"].shape == (3, rows, rank)
        for s, (r, a) in enumerate(files[2]):
            pair = a.get(f"blk.0.{stem}.weight")
            assert t["ranks"][s].item() == (0 if pair is None else r)
            if pair is not None:
                assert np.array_equal(t["A"][s, :r].numpy(), pair[0]) and np.array_equal(t["B"][s, :, :r].numpy(), pair[1])
                assert t["scales"][s].item() == pytest.approx({0: 2.0, 1: 0.5, 2: 1.0}[s])
            assert (t["A"][s, r if pair is not None else 0:] == 0).all()
    with pytest.raises(KeyError):
        loader.GGUFModel(files[0] / "model.gguf").q4k("blk.0.attn_q.weight.lora_a")


def test_rope_parameters_from_metadata(q4k, loader, files):
    p = loader.GGUFModel(files[0] / "model.gguf").rope(q4k, device="cpu")
    assert p["sections"] == (12, 10, 10) and p["layout"] == "adjacent" and p["order"] == "blocks"
    want = 50000.0 ** (-np.arange(32) / 32) / np.linspace(1, 4, 32, dtype=np.float32).astype(np.float64)
    assert np.allclose(p["inv_freq"].numpy(), want, rtol=1e-14)


def request_inputs(rng, C):
    hist = rng.integers(0, VOCAB, (C, 24)).astype(np.int32)
    off = np.arange(C + 1, dtype=np.int32) * 6
    words = (VOCAB + 31) // 32
    return dict(ids=rng.integers(-1, 3, C).astype(np.int32), pos=rng.integers(0, 5000, (3, C)).astype(np.int32), history=hist,
                history_len=rng.integers(0, 25, C).astype(np.int32),
                penalties=np.stack([np.full(C, 1.2), np.full(C, 0.1), np.full(C, 0.3)], 1).astype(np.float32),
                bias_tokens=rng.integers(0, VOCAB, 6 * C).astype(np.int32), bias_values=rng.integers(-8, 9, 6 * C).astype(np.float32),
                bias_offsets=off, mask=rng.integers(-2**31, 2**31, (2, words)).astype(np.int32),
                mask_rows=rng.integers(-1, 2, C).astype(np.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("C", [1, 5, 8])
def test_decode_step_of_requests(q4k, oracle, loader, files, C):
    import torch
    rng = np.random.default_rng(C)
    model = loader.GGUFModel(files[0] / "model.gguf")
    layer, adapters, rope = model.layer(0), load(loader, files), model.rope(q4k)
    head = model.to_device("output.weight").data
    groups = {key: grp for key, _, grp in loader.LLAMA_LAYER}
    ks = {"attn": 512, "o": 512, "ffn": 512, "down": 768}
    xs = {g: torch.empty((C, k), device="cuda") for g, k in ks.items()}
    outs = {key: torch.empty((C, layer[key].rows), device="cuda") for key in groups}
    xh = torch.empty((C, 512), device="cuda")
    req = {k: torch.from_numpy(v).cuda() for k, v in request_inputs(rng, C).items()}
    ws, ws_head = q4k.Workspace(1 << 22), q4k.Workspace(1 << 22)
    tasks = loader.layer_tasks(q4k, layer, xs, outs)
    lora = q4k.make_lora_tasks(loader.layer_adapter_items(adapters, 0, xs, outs))
    logits = torch.empty((C, VOCAB), device="cuda")

    def step():
        q4k.gemv_batch(tasks, C, ws)
        q4k.lora_batch(lora, req["ids"])
        q, k = (outs[n].view(C, -1, HEAD_DIM) for n in "qk")
        turned = q4k.rope_multi([q, k], req["pos"], out=[q, k], **rope)
        q4k.mul_mat_vec_q(head, xh, out=logits, ws=ws_head)
        picked = q4k.logits_process(logits, pick=True, **{n: req[n] for n in (
            "history", "history_len", "penalties", "bias_tokens", "bias_values", "bias_offsets", "mask", "mask_rows")})
        return turned, picked

    def fill(seed):
        r = np.random.default_rng(seed)
        x = {g: r.standard_normal((C, k)).astype(np.float32) for g, k in ks.items()}
        h = r.standard_normal((C, 512)).astype(np.float32)
        new = request_inputs(r, C)
        for g in ks:
            xs[g].copy_(torch.from_numpy(x[g]))
        xh.copy_(torch.from_numpy(h))
        for n, v in new.items():
            req[n].copy_(torch.from_numpy(v))
        return x, h, new

    def check(got, x, h, new):
        turned, (z, token, lse) = got
        inv = rope["inv_freq"].cpu().numpy()
        for key, grp in groups.items():
            name = {k: s for k, s, _ in loader.LLAMA_LAYER}[key]
            W = files[1][f"blk.0.{name}.weight"]
            base = oracle.gemv_f32(W, x[grp]).astype(np.float64)
            ad = adapters[f"blk.0.{name}.weight"]
            A, B = ad["A"].double().cpu().numpy(), ad["B"].double().cpu().numpy()
            want, mag = base.copy(), np.zeros_like(base)
            for j, a in enumerate(new["ids"]):
                if a >= 0:
                    s = float(ad["scales"][a])
                    want[j] += s * (B[a] @ (A[a] @ x[grp][j]))
                    mag[j] = abs(s) * (np.abs(B[a]) @ (np.abs(A[a]) @ np.abs(x[grp][j])))
            # the GEMV's bar, and sqrt(n) fp32 roundings of the adapter's terms
            tol = 1e-4 + 1e-5 * np.abs(base) + (SHAPES[name][1] + 17) ** 0.5 * 2.0 ** -24 * mag
            g = outs[key].double().cpu().numpy()
            if key in "qk":
                v = want.reshape(C, -1, HEAD_DIM)
                w, m = rope_reference(v, new["pos"], inv, rope["sections"], rope["layout"], rope["order"], 1.0)
                t = tol.reshape(v.shape)
                pair = np.stack([t[..., 0::2] + t[..., 1::2]] * 2, -1).reshape(t.shape)  # a turn mixes the errors of a pair
                want, tol = w.reshape(want.shape), (pair + 5 * 2.0 ** -24 * m).reshape(want.shape)
            assert (np.abs(g - want) <= tol).all(), (key, np.abs(g - want).max())
        raw = logits.cpu().numpy()
        o = oracle.gemv_f32(files[1]["output.weight"], h).astype(np.float64)
        assert (np.abs(raw - o) <= 1e-4 + 1e-5 * np.abs(o)).all()
        wz, wt, wl = logits_reference({"logits": raw, **{n: new[n] for n in new if n not in ("ids", "pos")}})
        assert np.array_equal(z.cpu().numpy(), wz) and np.array_equal(token.cpu().numpy(), wt)
        assert np.allclose(lse.cpu().numpy(), wl, rtol=0, atol=2e-5)

    data = fill(100)
    for _ in range(2):  # launches of the second step follow the first's closely
        got = step()
    torch.cuda.synchronize()
    check(got, *data)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in (101, 102):
        data = fill(seed)
        g.replay()
        torch.cuda.synchronize()
        check(got, *data)
    assert ws.status() == 0 and ws_head.status() == 0
