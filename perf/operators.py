"""The paged-cache and sampling operators: cases, plain forms and exact values.

Four operators that serve many sequences together: ``mfk_paged_append`` writes
new key/value rows into the pages of a cache, ``mfk_paged_gqa`` attends with
one new token per sequence over its pages, ``mfk_copy_pages`` copies pages
(the last page of a fork, a compaction) and ``mfk_sample`` draws the next
tokens.  ``run`` computes them in elementary torch operations, or through the
framework where ``own`` is set.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
WORKSPACE = 8 << 20


def listed():
    return [
        # One conversation: a single sequence's decode step, where launch latency is all of it.
        dict(name="attention one short", op="attention", seqs=1, low=257, high=257, q_heads=32, kv_heads=8, dim=64, page=16, dtype="f32"),
        # A batch of conversations of every age in the framework's F32 cache type.
        dict(name="attention ragged f32", op="attention", seqs=32, low=1, high=2320, q_heads=32, kv_heads=8, dim=64, page=16, dtype="f32"),
        # The large batched run: 512 sequences just past a 512-token prompt.
        dict(name="attention 512 bf16", op="attention", seqs=512, low=513, high=640, q_heads=32, kv_heads=8, dim=64, page=16, dtype="bf16"),
        # One very long document, the small model's heads: all of the work is the split over the length.
        dict(name="attention long f16", op="attention", seqs=1, low=131071, high=131071, q_heads=16, kv_heads=8, dim=64, page=64, dtype="f16"),
        # Wide heads in large groups, pages that are no power of two.
        dict(name="attention wide heads", op="attention", seqs=48, low=1000, high=5000, q_heads=16, kv_heads=2, dim=128, page=24, dtype="bf16"),
        # The decode step's write: one row for each of 512 sequences.
        dict(name="append decode", op="append", seqs=512, low=1, high=1, past=576, kv_heads=8, dim=64, page=16, dtype="bf16"),
        # Prompts of several lengths that enter the cache together.
        dict(name="append prompts", op="append", seqs=7, low=301, high=2501, past=100, kv_heads=8, dim=64, page=16, dtype="f32"),
        # Forks: the shared last page of a few sequences is copied in the six attention layers.
        dict(name="copy forks", op="copy", count=12, pages=600, layers=6, kv_heads=8, dim=64, page=16, dtype="bf16"),
        # Compaction of a cache after most of its sequences ended.
        dict(name="copy compaction", op="copy", count=1900, pages=4096, layers=6, kv_heads=8, dim=64, page=16, dtype="bf16"),
        # One conversation's next token with the usual filters.
        dict(name="sample one", op="sample", rows=1, width=65536, filters="all"),
        # The large batch: every row with its own settings.
        dict(name="sample 512", op="sample", rows=512, width=65536, filters="all"),
        # Temperature alone over an odd vocabulary.
        dict(name="sample odd width", op="sample", rows=33, width=32003, filters="none"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "copy", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64, rng.randint(1, 80)])
    kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 128, 8 * rng.randint(1, 16)])
    if op == "attention":
        seqs = _log_int(rng, 1, 512)
        token = 2 * kv_heads * dim * (4 if dtype == "f32" else 2)
        high = _log_int(rng, 2, max(2, min(131071, (256 << 20) // (token * seqs))))
        low = rng.choice([0, 1, high, rng.randint(0, high)])
        return dict(op=op, seqs=seqs, low=low, high=high, q_heads=kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if op == "append":
        seqs = _log_int(rng, 1, 512)
        high = _log_int(rng, 1, max(1, 8000 // seqs))
        return dict(op=op, seqs=seqs, low=rng.choice([0, 1, high]), high=high, past=rng.randint(0, 300), kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if op == "copy":
        layers = rng.randint(1, 8)
        page_bytes = 2 * layers * kv_heads * page * dim * (4 if dtype == "f32" else 2)
        count = _log_int(rng, 1, max(1, min(4000, (256 << 20) // page_bytes)))
        return dict(op=op, count=count, pages=2 * count + rng.randint(0, 50), layers=layers, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    width = _log_int(rng, 2, 200000)
    rows = _log_int(rng, 1, max(1, min(512, 32000000 // width)))
    return dict(op=op, rows=rows, width=width, filters=rng.choice(["all", "none", "top_k", "top_p", "min_p"]))


def _lengths(case):
    """The lengths of a case's sequences: spread over [low, high], the same for every seed."""
    span = case["high"] - case["low"] + 1
    return [case["low"] + (((i + 1) * 2654435761 % (1 << 32)) * span >> 32) for i in range(case["seqs"])]


def _page_tables(lengths, page, generator):
    """A page table for the lengths whose pages lie in no order, and the number of pages."""
    need = np.array([-(-n // page) for n in lengths], np.int64)
    most, pages = max(1, int(need.max())), int(need.sum()) + 3
    order = torch.randperm(pages, generator=generator).numpy().astype(np.int32)
    table = np.full((len(lengths), most), -1, np.int32)
    table[np.arange(most) < need[:, None]] = order[: int(need.sum())]
    return torch.from_numpy(table).cuda(), pages


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gpu, device="cuda", dtype=dtype)

    s = dict(case)
    if case["op"] in ("attention", "append"):
        lengths = _lengths(case)
        h, d, dtype = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
        past = [case.get("past", 0) + i % 5 for i in range(len(lengths))] if case["op"] == "append" else [0] * len(lengths)
        s["table"], pages = _page_tables([n + p for n, p in zip(lengths, past)], case["page"], host)
        s["keys"], s["values"] = (normal(pages, h, case["page"], d, dtype=dtype) for _ in range(2))
        if case["op"] == "attention":
            # Normalised queries and keys: their scores spread as a trained model's do.
            s["q"] = normal(len(lengths), case["q_heads"] * d) * 2.0
            s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
            s["out"] = torch.empty_like(s["q"])
            s["workspace"] = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
        else:
            total = sum(lengths)
            s["k"], s["v"] = normal(total, h * d), normal(total, h * d)
            s["starts"] = torch.tensor(past, dtype=torch.int32, device="cuda")
            s["offsets"] = torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32, device="cuda")
    elif case["op"] == "copy":
        s["pools"] = normal(2 * case["layers"], case["pages"], case["kv_heads"], case["page"], case["dim"], dtype=DTYPES[case["dtype"]])
        order = torch.randperm(case["pages"], generator=host).numpy().astype(np.uint32)
        s["sources"], s["targets"] = order[: case["count"]].copy(), order[case["count"] : 2 * case["count"]].copy()
    else:
        rows, width = case["rows"], case["width"]
        logits = normal(rows, width) * 2.0
        # A few likely tokens above a broad floor.
        likely = torch.randint(0, width, (rows, 24), generator=gpu, device="cuda")
        s["logits"] = logits.scatter_add_(1, likely, 4.0 - 3.0 * torch.log(torch.rand(rows, 24, generator=gpu, device="cuda").clamp_min(1e-3)))

        def spread(*values):
            at = torch.randint(0, len(values), (rows,), generator=host)
            return torch.tensor(values)[at].cuda()

        s["uniform"] = torch.rand(rows, generator=gpu, device="cuda")
        s["temperature"] = spread(0.6, 0.8, 1.0, 1.3)
        some = case["filters"]
        s["top_k"] = spread(20, 50, 200, 0).to(torch.int32) if some in ("all", "top_k") else None
        s["top_p"] = spread(0.8, 0.9, 0.95, 1.0) if some in ("all", "top_p") else None
        s["min_p"] = spread(0.0, 0.02, 0.05, 0.1) if some in ("all", "min_p") else None
        s["out"] = torch.empty(rows, device="cuda")
    return s


def _attention(s):
    n, h, d, page = s["seqs"], s["kv_heads"], s["dim"], s["page"]
    table = s["table"].clamp_min(0).long()
    seen = torch.arange(table.shape[1] * page, device="cuda") < s["lengths"][:, None]

    def rows(pages):  # [n, h, tokens, d]
        x = pages[table].float().permute(0, 2, 1, 3, 4).reshape(n, h, -1, d)
        return torch.where(seen[:, None, :, None], x, 0.0)

    q = s["q"].view(n, h, -1, d)
    scores = (q @ rows(s["keys"]).transpose(2, 3)) * d**-0.5
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    most = scores.amax(3, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(most), most, 0.0))
    total = p.sum(3, keepdim=True)
    out = (p @ rows(s["values"])) / torch.where(total > 0, total, 1.0)
    return out.reshape(n, -1)


def _append(s):
    offsets = s["offsets"].long()
    row = torch.arange(s["k"].shape[0], device="cuda")
    seq = torch.searchsorted(offsets, row, right=True) - 1
    position = s["starts"][seq] + row - offsets[seq]
    at = s["table"][seq, position // s["page"]].long()
    for pages, rows in ((s["keys"], s["k"]), (s["values"], s["v"])):
        pages[at, :, position % s["page"]] = rows.view(-1, s["kv_heads"], s["dim"]).to(pages.dtype)
    return s["keys"], s["values"]


def _copy(s):
    sources, targets = (torch.from_numpy(s[n].astype(np.int64)).cuda() for n in ("sources", "targets"))
    s["pools"][:, targets] = s["pools"][:, sources]
    return s["pools"]


def _sample(s):
    x = s["logits"].double()
    rows, width = x.shape
    weight = torch.exp((x - x.amax(1, keepdim=True)) / s["temperature"].double()[:, None])
    order = torch.sort(s["logits"], dim=1, descending=True, stable=True).indices
    ordered = weight.gather(1, order)
    keep = torch.ones_like(ordered, dtype=torch.bool)
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"], width)
        keep &= torch.arange(width, device="cuda") < k[:, None]
    if s["top_p"] is not None:
        inside = torch.where(keep, ordered, 0.0)
        mass = inside.cumsum(1)
        keep &= (mass - inside < s["top_p"].double()[:, None] * mass[:, -1:]) | (s["top_p"][:, None] >= 1.0)
        keep[:, 0] = True
    if s["min_p"] is not None:
        keep &= (ordered >= s["min_p"].double()[:, None]) | (ordered == 1.0)
    kept = torch.zeros_like(weight).scatter_(1, order, torch.where(keep, ordered, 0.0))
    mass = kept.cumsum(1)
    return (mass <= s["uniform"].double()[:, None] * mass[:, -1:]).sum(1).float()


def run(s):
    if not own:
        return {"attention": _attention, "append": _append, "copy": _copy, "sample": _sample}[s["op"]](s)
    from runtime_b200 import _lib
    from runtime_b200.backend import _check

    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream

    def at(name):
        return None if s[name] is None else s[name].data_ptr()

    if s["op"] == "attention":
        _check(lib.mfk_paged_gqa(at("out"), at("q"), at("keys"), at("values"), CODES[s["dtype"]], s["keys"].shape[0], s["page"], at("table"), s["table"].shape[0], s["table"].shape[1], at("lengths"), None, s["seqs"], s["q_heads"], s["kv_heads"], s["dim"], at("workspace"), WORKSPACE, stream))
        return s["out"]
    if s["op"] == "append":
        _check(lib.mfk_paged_append(at("keys"), at("values"), CODES[s["dtype"]], s["keys"].shape[0], s["page"], at("table"), s["table"].shape[0], s["table"].shape[1], at("k"), at("v"), s["k"].shape[0], at("starts"), at("offsets"), None, s["seqs"], s["kv_heads"], s["dim"], stream))
        return s["keys"], s["values"]
    if s["op"] == "copy":
        pools = s["pools"]
        page_bytes = pools[0, 0].numel() * pools.element_size()
        bases = np.arange(pools.shape[0], dtype=np.uint64) * np.uint64(page_bytes * pools.shape[1]) + np.uint64(pools.data_ptr())
        _check(lib.mfk_copy_pages(bases.ctypes.data, pools.shape[0], pools.shape[1], page_bytes, s["sources"].ctypes.data, s["targets"].ctypes.data, s["count"], stream))
        return pools
    _check(lib.mfk_sample(at("out"), at("logits"), s["rows"], s["width"], at("temperature"), at("top_k"), at("top_p"), at("min_p"), at("uniform"), stream))
    return s["out"]


def work(case):
    if case["op"] == "sample":
        # Every logit once; its weight and the running mass.
        return {"bytes": case["rows"] * (4.0 * case["width"] + 24), "flops": 4.0 * case["rows"] * case["width"]}
    size = 4 if case["dtype"] == "f32" else 2
    row = case["kv_heads"] * case["dim"]
    if case["op"] == "copy":
        return {"bytes": 4.0 * case["layers"] * case["count"] * case["page"] * row * size, "flops": 0.0}
    lengths = _lengths(case)
    tokens = sum(lengths)
    if case["op"] == "append":
        return {"bytes": 2.0 * tokens * row * (4 + size) + 12.0 * len(lengths), "flops": 0.0}
    table = sum(-(-n // case["page"]) for n in lengths)
    wide = case["q_heads"] * case["dim"]
    return {"bytes": 2.0 * tokens * row * size + 8.0 * len(lengths) * wide + 4.0 * (table + len(lengths)), "flops": 4.0 * tokens * wide}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        return None
    if case["op"] == "sample":
        ids = []
        for r in range(case["rows"]):
            x = s["logits"][r].cpu().numpy().astype(np.float64)
            t, u, k, p, m = (None if s[n] is None else float(s[n][r]) for n in ("temperature", "uniform", "top_k", "top_p", "min_p"))
            w = np.exp((x - x.max()) / t)
            first = np.lexsort((np.arange(x.size), -x))
            if k:
                first = first[: int(k)]
            if p is not None and p < 1.0:
                before = np.concatenate(([0.0], np.cumsum(w[first])))
                first = first[: max(1, int(np.searchsorted(before[:-1], p * before[-1], side="left")))]
            if m:
                first = first[w[first] >= m]
            first = np.sort(first)
            mass = np.cumsum(w[first])
            ids.append(float(first[np.searchsorted(mass, u * mass[-1], side="right")]))
        return np.array(ids)
    page, h, d = case["page"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        result = [s["keys"].double(), s["values"].double()]
        row = 0
        for i, n in enumerate(_lengths(case)):
            position = torch.arange(n, device="cuda") + int(s["starts"][i])
            where = s["table"][i, torch.div(position, page, rounding_mode="floor")].long()
            for pages, rows in zip(result, (s["k"], s["v"])):
                pages[where, :, position % page] = rows[row : row + n].double().view(n, h, d)
            row += n
        return tuple(result)
    out = torch.zeros(case["seqs"], case["q_heads"], d, dtype=torch.float64, device="cuda")
    for i, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        where = s["table"][i, : -(-n // page)].long()
        k, v = (s[x][where].transpose(0, 1).reshape(h, -1, d)[:, :n].double() for x in ("keys", "values"))
        q = s["q"][i].double().view(h, -1, d)
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(d), 2)
        out[i] = torch.einsum("hgn,hnd->hgd", p, v).reshape(-1, d)
    return out.view(case["seqs"], -1)
