"""The operators that a batch of requests needs around its shared projections, measured over their real range.

lora    low-rank adapters of many requests beside a shared projection (lora_add, lora_batch)
rope    rotary positions with several axes on the query and key outputs (rope_multi)
logits  penalties, biases and grammar masks on the head's logits, the greedy token and log-sum-exp (logits_process)
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def package():
    """The framework's package: its folder's name is no identifier, so it is loaded by path."""
    if "q4k_b200" not in sys.modules:
        folder = Path.cwd() / "gemv-q4_k-optimization_b200"
        spec = importlib.util.spec_from_file_location("q4k_b200", folder / "__init__.py",
                                                      submodule_search_locations=[str(folder)])
        module = importlib.util.module_from_spec(spec)
        sys.modules["q4k_b200"] = module
        spec.loader.exec_module(module)
    return sys.modules["q4k_b200"]


def ints(text):
    return [int(t) for t in str(text).split(",")]


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one request decodes through one adapted 4096 x 4096 projection: nothing but latency
        dict(name="lora_one", op="lora", cols=1, K=4096, rows="4096", rank=16, slots=8, used=1, type="bfloat16",
             ragged=False, order="mixed"),
        # eight requests, each with an adapter and a rank of its own, through q, k and v in one call; one has none
        dict(name="lora_qkv_8", op="lora", cols=8, K=4096, rows="4096,1024,1024", rank=64, slots=16, used=8,
             type="float16", ragged=True, order="mixed"),
        # the long reduction of the down projection, adapters kept in 32 bits
        dict(name="lora_down_8", op="lora", cols=8, K=14336, rows="4096", rank=32, slots=4, used=3, type="float32",
             ragged=False, order="mixed"),
        # a wide decode batch over the adapters of a busy server
        dict(name="lora_batch_64", op="lora", cols=64, K=4096, rows="14336", rank=32, slots=32, used=16,
             type="bfloat16", ragged=True, order="mixed"),
        # prompts of several requests in one batch, odd in every size
        dict(name="lora_prompt_odd", op="lora", cols=777, K=1000, rows="2049", rank=24, slots=6, used=4,
             type="float16", ragged=True, order="runs"),
        # long prompts of three requests
        dict(name="lora_prompt_4096", op="lora", cols=4096, K=4096, rows="4096", rank=64, slots=8, used=3,
             type="bfloat16", ragged=False, order="runs"),
        # the queries and keys of a decode step, text and image positions, behind a long history
        dict(name="rope_decode_8", op="rope", cols=8, heads="32,8", dim=128, rot=128, sections="16,24,24",
             order="blocks", layout="half", base=1e6, far=131072, out="float32"),
        # part of each head rotated, neighbouring pairs, an odd number of columns, half-width output for a cache
        dict(name="rope_partial_1001", op="rope", cols=1001, heads="20,4", dim=96, rot=64, sections="12,10,10",
             order="interleaved", layout="adjacent", base=1e4, far=32768, out="float16"),
        # a long prompt with video frames
        dict(name="rope_prompt_8192", op="rope", cols=8192, heads="32,8", dim=128, rot=128, sections="24,20,20",
             order="interleaved", layout="half", base=5e6, far=262144, out="float32"),
        # one request, the usual short penalty window, no grammar
        dict(name="logits_one", op="logits", cols=1, vocab=32000, history=64, bias=0, masked=0.0, allow=1.0),
        # eight requests of a large vocabulary, half of them under a grammar that allows few tokens
        dict(name="logits_8", op="logits", cols=8, vocab=128256, history=512, bias=300, masked=0.5, allow=0.002),
        # the rows of a large batch, long windows, an odd vocabulary
        dict(name="logits_rows_384", op="logits", cols=384, vocab=128257, history=1024, bias=64, masked=0.25,
             allow=0.5),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw_one(rng):
    op = rng.choice(["lora", "rope", "logits"])
    if op == "lora":
        step = rng.choice([1, 8, 64])
        cols = log_int(rng, 1, 4096)
        slots = log_int(rng, 1, 32)
        rows = [step * log_int(rng, max(1, 64 // step), 14336 // step) for _ in range(rng.choice([1, 1, 2, 3]))]
        return dict(op=op, cols=cols, K=step * log_int(rng, max(1, 64 // step), 14336 // step),
                    rows=",".join(map(str, rows)), rank=log_int(rng, 1, 128), slots=slots,
                    used=rng.randint(1, slots), type=rng.choice(sorted(TYPES)), ragged=rng.random() < 0.5,
                    order=rng.choice(["mixed", "runs"]))
    if op == "rope":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        rot = rng.choice([dim, dim, dim // 2])
        half = rot // 2
        axes = rng.choice([1, 2, 3, 3, 4])
        cut = sorted(rng.sample(range(1, half), axes - 1))
        heads = rng.choice(["32,8", "8,2", "20,4", "7,1", "16"])
        return dict(op=op, cols=log_int(rng, 1, 8192), heads=heads, dim=dim, rot=rot,
                    sections=",".join(str(b - a) for a, b in zip([0] + cut, cut + [half])),
                    order=rng.choice(["blocks", "interleaved"]), layout=rng.choice(["half", "adjacent"]),
                    base=rng.choice([1e4, 5e5, 1e6]), far=log_int(rng, 16, 1 << 20),
                    out=rng.choice(sorted(TYPES)))
    return dict(op=op, cols=log_int(rng, 1, 512), vocab=log_int(rng, 1000, 256000),
                history=rng.choice([0, log_int(rng, 1, 4096)]), bias=rng.choice([0, log_int(rng, 1, 512)]),
                masked=rng.choice([0.0, 0.25, 0.5, 1.0]), allow=rng.choice([0.0005, 0.02, 0.5, 0.98]))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = max(most.get(c["op"], 0), w["bytes"])
    c = draw_one(rng)
    while work(c)["bytes"] > most[c["op"]]:
        c = draw_one(rng)
    return c


def work(case):
    if case["op"] == "lora":
        C, K, S = case["cols"], case["K"], case["used"]
        rank = case["rank"] * (0.5 if case["ragged"] else 1.0)  # ragged ranks spread over 1..rank
        size = 4 if case["type"] == "float32" else 2
        rows = ints(case["rows"])
        own_slots = min(S, C)
        bytes_, flops = 4 * C * K, 0
        for N in rows:
            bytes_ += 8 * C * N + own_slots * rank * (K + N) * size
            flops += 2 * C * rank * (K + N)
        return {"bytes": bytes_, "flops": flops}
    if case["op"] == "rope":
        n = case["cols"] * sum(ints(case["heads"])) * case["dim"]
        size = 4 if case["out"] == "float32" else 2
        return {"bytes": n * (4 + size) + case["cols"] * 4 * len(ints(case["sections"])), "flops": 3 * n}
    C, V = case["cols"], case["vocab"]
    # of a masked row only the 32-byte sectors (8 tokens) that hold an allowed token have to be read
    touched = 1 - (1 - case["allow"]) ** 8
    read = C * V * 4 * (1 - case["masked"] + case["masked"] * touched)
    lists = C * (case["history"] * 4 + case["bias"] * 8) + C * case["masked"] * V / 8
    return {"bytes": read + C * V * 4 + lists, "flops": 4 * C * V}


# ---------------------------------------------------------------------------
# what a user's program has in hand
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    def whole(lo, hi, *shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, device="cuda", generator=g, dtype=dtype)

    s = {"op": case["op"], "case": dict(case)}
    C = case["cols"]
    if case["op"] == "lora":
        K, S, R, t = case["K"], case["slots"], case["rank"], TYPES[case["type"]]
        s["x"] = normal(C, K)
        s["x"][:, :: max(1, K // 7)] *= 20.0  # the few large channels of a hidden state
        rows = ints(case["rows"])
        s["A"] = [(normal(S, R, K) / math.sqrt(K)).to(t) for _ in rows]
        s["B"] = [(normal(S, N, R) / math.sqrt(R)).to(t) for N in rows]
        s["base"] = [normal(C, N) for N in rows]
        s["scales"] = torch.rand(S, device="cuda", generator=g) + 0.25
        s["ranks"] = whole(1, R + 1, S) if case["ragged"] else torch.full((S,), R, device="cuda", dtype=torch.int32)
        used = torch.randperm(S, device="cuda", generator=g)[: case["used"]].to(torch.int32)
        pick = whole(0, case["used"], C).sort().values if case["order"] == "runs" else whole(0, case["used"], C)
        if case["order"] == "mixed" and case["used"] >= C:
            pick = torch.randperm(case["used"], device="cuda", generator=g)[:C]
        s["ids"] = used[pick.long()]
        if C >= 8 and case["order"] == "mixed":
            s["ids"][5] = -1  # a request without an adapter
        return s
    if case["op"] == "rope":
        D, rot = case["dim"], case["rot"]
        s["x"] = [normal(C, H, D) for H in ints(case["heads"])]
        s["sections"] = tuple(ints(case["sections"]))
        # text runs (all axes alike) with a frame of patches in between, up to the far end of a long history
        start = max(0, case["far"] - C)
        run = torch.arange(C, device="cuda", dtype=torch.int32) + int(start * ((seed % 7) + 1) / 7)
        pos = run.repeat(len(s["sections"]), 1)
        lo, hi = C // 4, C // 4 + C // 2
        side = max(1, math.isqrt(max(1, hi - lo)))
        k = torch.arange(hi - lo, device="cuda", dtype=torch.int32)
        patch = [k // (side * side), k // side, k % side, k % 3]
        for a in range(len(s["sections"])):
            pos[a, lo:hi] = run[lo : lo + 1] + patch[a]
        s["pos"] = pos.contiguous()
        i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
        s["inv_freq"] = torch.exp(-(2.0 * i / rot) * math.log(case["base"]))
        return s
    V, L, nb = case["vocab"], case["history"], case["bias"]
    s["logits"] = normal(C, V) * 3.0
    s["history"] = whole(0, V, C, max(1, L))
    if L > 8:
        s["history"][:, : L // 2] = s["history"][:, : L // 2] % max(1, V // 50)  # frequent tokens come again
    s["history_len"] = whole(0, L + 1, C) if L else torch.zeros(C, device="cuda", dtype=torch.int32)
    pen = torch.rand((C, 3), device="cuda", generator=g)
    s["penalties"] = torch.stack([1.0 + 0.5 * pen[:, 0], pen[:, 1], pen[:, 2] - 0.25], 1).contiguous()
    s["bias_tokens"] = s["bias_values"] = s["bias_offsets"] = None
    if nb:
        lens = whole(0, nb + 1, C, dtype=torch.int64)
        off = torch.zeros(C + 1, device="cuda", dtype=torch.int64)
        off[1:] = lens.cumsum(0)
        total = C * nb  # room for the longest lists; the offsets say how much of it is used
        s["bias_tokens"] = whole(0, V, total)
        # eighths: sums of repeated entries are exact in any order; a banned token now and then
        s["bias_values"] = whole(-40, 41, total).float() / 8.0
        s["bias_values"][::97] = -math.inf
        s["bias_offsets"] = off.to(torch.int32)
    s["mask"] = s["mask_rows"] = None
    m = int(round(case["masked"] * C))
    if m:
        words = (V + 31) // 32
        bits = torch.rand((m, words * 32), device="cuda", generator=g) < case["allow"]
        w = (bits.view(m, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
        s["mask"] = torch.where(w >= 2**31, w - 2**32, w).to(torch.int32).contiguous()
        rows = torch.full((C,), -1, device="cuda", dtype=torch.int32)
        at = torch.randperm(C, device="cuda", generator=g)[:m]
        rows[at] = torch.arange(m, device="cuda", dtype=torch.int32)
        s["mask_rows"] = rows
        if m > 2:
            s["mask"][1] = 0  # a grammar that is at its end allows nothing
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return {"lora": run_lora, "rope": run_rope, "logits": run_logits}[s["op"]](s)


def run_lora(s):
    if own:
        q = package()
        if len(s["A"]) == 1:
            return [q.lora_add(s["x"], s["A"][0], s["B"][0], s["ids"], base=s["base"][0], ranks=s["ranks"],
                               scales=s["scales"])]
        return q.lora_batch([dict(x=s["x"], A=a, B=b, base=y, ranks=s["ranks"], scales=s["scales"])
                             for a, b, y in zip(s["A"], s["B"], s["base"])], s["ids"])
    return [plain_lora(s["x"], a, b, y, s["ids"], s["ranks"], s["scales"])
            for a, b, y in zip(s["A"], s["B"], s["base"])]


def plain_lora(x, A, B, base, ids, ranks, scales):
    S, R, K = A.shape
    N = B.shape[1]
    # every column against every slot's rows in one product, then only its own slot's are kept
    u = x @ A.float().reshape(S * R, K).T
    slot = torch.arange(S, device=x.device).repeat_interleave(R)
    t = torch.arange(R, device=x.device).repeat(S)
    keep = (ids[:, None] == slot[None, :]) & (t < ranks.long()[slot])[None, :]
    u = torch.where(keep, u * scales[slot], torch.zeros((), device=x.device))
    return base + u @ B.float().permute(0, 2, 1).reshape(S * R, N)


def run_rope(s):
    c = s["case"]
    out = TYPES[c["out"]]
    if own:
        return package().rope_multi(s["x"], s["pos"], s["inv_freq"], s["sections"], layout=c["layout"],
                                    order=c["order"], dtype=out)
    axis = pair_axes(s["sections"], c["order"], s["inv_freq"].numel(), s["pos"].device)
    angle = s["pos"][axis].T.double() * s["inv_freq"]  # (columns, pairs); far positions need 64 bits
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    return [plain_rope(x, cos, sin, c["rot"], c["layout"], out) for x in s["x"]]


def pair_axes(sections, order, pairs, device):
    """The axis of each pair. blocks: the axes' sections one after another, repeated; interleaved: the axes in turn
    for as long as each has pairs left, the others going to the first axis."""
    n = len(sections)
    i = torch.arange(pairs, device=device)
    if order == "blocks":
        ends = torch.tensor(sections, device=device).cumsum(0)
        return torch.searchsorted(ends, i % ends[-1], right=True)
    size = torch.tensor(sections, device=device)
    turn = i % n
    return torch.where(i // n < size[turn], turn, torch.zeros_like(turn))


def plain_rope(x, cos, sin, rot, layout, out):
    half = rot // 2
    if layout == "half":
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1).to(out)


def run_logits(s):
    if own:
        return list(package().logits_process(
            s["logits"], history=s["history"], history_len=s["history_len"], penalties=s["penalties"],
            bias_tokens=s["bias_tokens"], bias_values=s["bias_values"], bias_offsets=s["bias_offsets"],
            mask=s["mask"], mask_rows=s["mask_rows"], pick=True))
    z = s["logits"]
    C, V = z.shape
    dev = z.device
    if s["bias_tokens"] is not None:
        off = s["bias_offsets"].long()
        at = torch.arange(s["bias_tokens"].numel(), device=dev)
        col = torch.searchsorted(off, at, right=True) - 1
        live = at < off[-1]
        dense = torch.zeros((C, V), device=dev)
        dense.index_put_((col.clamp(max=C - 1), s["bias_tokens"].long()),
                         torch.where(live, s["bias_values"], torch.zeros((), device=dev)), accumulate=True)
        z = z + dense
    live = torch.arange(s["history"].shape[1], device=dev)[None, :] < s["history_len"][:, None]
    count = torch.zeros((C, V), device=dev).scatter_add_(1, s["history"].long(), live.float())
    rep, freq, here = s["penalties"][:, :1], s["penalties"][:, 1:2], s["penalties"][:, 2:]
    z = torch.where(count > 0, torch.where(z > 0, z / rep, z * rep) - (count * freq + here), z)
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=dev)) & 1
        bits = bits.reshape(bits.shape[0], -1)[:, :V].bool()
        allowed = bits[s["mask_rows"].long().clamp(min=0)] | (s["mask_rows"] < 0)[:, None]
        z = torch.where(allowed, z, torch.full((), -math.inf, device=dev))
    top, token = z.max(-1)
    none = top == -math.inf
    token = torch.where(none, torch.full_like(token, -1), token).to(torch.int32)
    shift = torch.where(none, torch.zeros_like(top), top)
    lse = shift + torch.log(torch.exp(z - shift[:, None]).sum(-1))
    return [z, token, lse]


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lora":
        out = []
        for A, B, base in zip(s["A"], s["B"], s["base"]):
            y = base.double()
            for a in torch.unique(s["ids"]).tolist():
                if a < 0:
                    continue
                r = int(s["ranks"][a])
                mine = (s["ids"] == a).nonzero()[:, 0]
                u = s["x"][mine].double() @ A[a, :r].double().T
                y[mine] += float(s["scales"][a].double()) * (u @ B[a, :, :r].double().T)
            out.append(y)
        return out
    if case["op"] == "rope":
        n, half = len(s["sections"]), case["rot"] // 2
        if case["order"] == "blocks":
            one = [a for a, k in enumerate(s["sections"]) for _ in range(k)]
            axis = [one[i % len(one)] for i in range(half)]
        else:
            axis = [i % n if i // n < s["sections"][i % n] else 0 for i in range(half)]
        lo = [i if case["layout"] == "half" else 2 * i for i in range(half)]
        hi = [i + half if case["layout"] == "half" else 2 * i + 1 for i in range(half)]
        phi = torch.stack([s["pos"][axis[i]].double() * s["inv_freq"][i] for i in range(half)], 1)[:, None, :]
        out = []
        for x in s["x"]:
            v = x.double()
            y = v.clone()
            y[..., lo] = v[..., lo] * phi.cos() - v[..., hi] * phi.sin()
            y[..., hi] = v[..., hi] * phi.cos() + v[..., lo] * phi.sin()
            out.append(y)
        return out
    C, V = s["logits"].shape
    z, lse = s["logits"].double(), torch.empty(C, device="cuda", dtype=torch.float64)
    length, rows = s["history_len"].tolist(), s["mask_rows"].tolist() if s["mask"] is not None else [-1] * C
    off = s["bias_offsets"].tolist() if s["bias_offsets"] is not None else None
    bit = torch.arange(32, device="cuda")
    for j in range(C):
        if off is not None:
            k = slice(off[j], off[j + 1])
            z[j].index_add_(0, s["bias_tokens"][k].long(), s["bias_values"][k].double())
        seen, times = torch.unique(s["history"][j, : length[j]].long(), return_counts=True)
        r, f, p = (s["penalties"][j, i].double() for i in range(3))
        v = z[j, seen]
        z[j, seen] = torch.where(v > 0, v / r, v * r) - (times.double() * f + p)
        if rows[j] >= 0:
            gone = ((s["mask"][rows[j]][:, None] >> bit) & 1).flatten()[:V] == 0
            z[j, gone] = -math.inf
        lse[j] = torch.logsumexp(z[j], 0)
    return [z, None, lse]
